"""Expert row routing at the ends of what its calls allow."""
import pytest
import torch

from geeps_amd import routing


def padding_starts(places, end):
    """The first place that each of a wave's 64 lanes clears behind `places` rows of a group that ends at `end`,
    as 32-bit signed and as unsigned arithmetic have it."""
    signed = [(places + lane + 2 ** 31) % 2 ** 32 - 2 ** 31 for lane in range(64)]
    return [p for p in signed if p < end], [p for p in range(places, places + 64) if p < end]


def test_most_rows_pass_31_bits():
    """Why the test below has these sizes: some lanes' places behind the last group pass 2^31, and as signed
    numbers they would lie before the group's end, and before the map."""
    tokens, align = (1 << 31) - 40, 32
    rows = routing.group_rows(tokens, 1, 1, align)
    assert rows == (1 << 31) - 32 == -(-tokens // align) * align
    signed, unsigned = padding_starts(tokens, rows)
    assert min(signed) < 0 and unsigned == list(range(tokens, rows))


@pytest.mark.gpu
def test_padding_of_the_most_rows(dev):
    tokens, align = (1 << 31) - 40, 32
    rows = routing.group_rows(tokens, 1, 1, align)
    ids = torch.zeros(tokens, 1, dtype=torch.int32, device=dev)
    route = routing.sort_tokens(ids, 1, align)
    assert route.counts.tolist() == [tokens] and route.offsets.tolist() == [0, rows]
    del ids
    want = torch.arange(tokens, dtype=torch.int32, device=dev)
    assert torch.equal(route.position.view(-1), want)
    assert torch.equal(route.order[:tokens], want)
    assert route.order[tokens:].tolist() == [-1] * (rows - tokens)
