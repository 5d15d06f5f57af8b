"""beam_reorder: ranks and lengths of 64 bits, states that lie between each other in one buffer, and waves with few columns."""
import pytest
import torch

pytestmark = pytest.mark.gpu

I31, I32, I63 = 1 << 31, 1 << 32, (1 << 63) - 1


RANKS = {
    "int64": torch.tensor([[0, 1, 2, 3, I31 - 1, I31, I32, I32 + 1, I63, -1, -I31 - 5, -I63]]).repeat(3, 1),
    "int32": torch.tensor([[0, 1, 2, 3, I31 - 1, I31 - 2, 7, 8, -1, -2, -I31, 5]]).repeat(3, 1).to(torch.int32),
    "none": None,
}
LENGTHS = {
    "int": 3, "negative": -2, "int_31": I31, "int_40": 1 << 40, "int_63": I63,
    "int64": torch.tensor([2, I63, I32]), "int64_too": torch.tensor([-I63, I31, I32 + 2]),
    "int32": torch.tensor([2, I31 - 1, -1]).to(torch.int32),
}


@pytest.mark.parametrize("rank", list(RANKS))
@pytest.mark.parametrize("length", list(LENGTHS))
def test_ranks_and_lengths_compare_in_64_bits(rank, length):
    import mpnn_amd
    from oracle import beam_oracle as orc

    g = torch.Generator().manual_seed(1)
    rank, length = RANKS[rank], LENGTHS[length]
    parent = torch.tensor([[2, 0, 1], [1, 1, 0], [0, 2, 2]])
    cpu = [torch.randn(3, 3, 12, 8, generator=g), torch.randint(0, 99, (3, 3, 12), generator=g)]
    gpu = [x.cuda() for x in cpu]
    cuda = lambda x: x.cuda() if isinstance(x, torch.Tensor) else x   # noqa: E731
    mpnn_amd.beam_reorder(gpu, parent.cuda(), cuda(length), cuda(rank))
    rank = rank if rank is None else rank.long()        # torch compares a 32-bit tensor with a number in 32 bits
    for x, y in zip(cpu, gpu):
        same = torch.equal(y.cpu(), orc.reorder(x, parent, length, rank))
        assert same


def test_rank_that_lies_in_a_state():
    """A 64-bit rank is compared before any state moves."""
    import mpnn_amd
    from oracle import beam_oracle as orc

    g = torch.Generator().manual_seed(2)
    table = torch.randint(0, 9, (2, 2, 9), generator=g)
    parent = torch.tensor([[1, 0], [1, 1]])
    dev = table.cuda()
    mpnn_amd.beam_reorder(dev, parent.cuda(), length=4, rank=dev[:, 0])
    assert torch.equal(dev.cpu(), orc.reorder(table, parent, 4, table[:, 0]))


def test_64_bit_rank_in_a_graph():
    """The comparison is part of the captured call: replays follow the rank, the length and the parents of the day."""
    import mpnn_amd
    from oracle import beam_oracle as orc

    g = torch.Generator().manual_seed(5)
    new = lambda: (torch.randn(2, 3, 12, 8, generator=g), torch.randint(0, 3, (2, 3), generator=g),   # noqa: E731
                   torch.randint(0, 12, (2,), generator=g), torch.argsort(torch.rand(2, 12, generator=g), 1))
    state, parent, length, rank = (x.cuda() for x in new())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mpnn_amd.beam_reorder(state, parent, length, rank)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mpnn_amd.beam_reorder(state, parent, length, rank)
    for _ in range(4):
        cpu = new()
        for x, y in zip((state, parent, length, rank), cpu):
            x.copy_(y)
        graph.replay()
        same = torch.equal(state.cpu(), orc.reorder(*cpu))
        assert same


@pytest.mark.parametrize("W", [65, 66, 100, 128, 129, 200, 255, 256])
@pytest.mark.parametrize("columns", [1, 3, 63, 64, 65, 130])
def test_waves_with_few_columns(W, columns):
    """Beyond 64 beams every lane holds the parents of its beams, also a lane without a column, or whose position stays."""
    import mpnn_amd
    from oracle import beam_oracle as orc

    g = torch.Generator().manual_seed(W + columns)
    parent = torch.randint(0, W, (2, W), generator=g)
    cpu = torch.randn(2, W, columns, generator=g)
    dev = cpu.cuda()
    mpnn_amd.beam_reorder(dev, parent.cuda())
    want = orc.reorder(cpu, parent)
    assert torch.equal(dev.cpu(), want)
    rank = torch.argsort(torch.rand(2, columns, generator=g), 1).to(torch.int32)
    length = torch.tensor([1, columns // 2])
    mpnn_amd.beam_reorder(dev, parent.cuda(), length.cuda(), rank.cuda())
    assert torch.equal(dev.cpu(), orc.reorder(want, parent, length, rank))


PACKED = {   # views of one buffer that share no byte
    "keys_values_prefix": ((2, 3, 2, 4, 9, 8), lambda x: [x[:, :, 0, :, :5], x[:, :, 1, :, :5]], None),
    "keys_values": ((2, 3, 2, 4, 9, 8), lambda x: [x[:, :, 1], x[:, :, 0]], None),
    "behind_heads": ((2, 3, 4, 2, 9, 8), lambda x: [x[:, :, :, 0, :5], x[:, :, :, 1, :5]], None),
    "layers": ((2, 3, 3, 2, 9, 8), lambda x: [x[:, :, i, j, :6] for i in range(3) for j in range(2)], None),
    "different_lengths": ((2, 3, 2, 4, 9, 8), lambda x: [x[:, :, 0, :, :5], x[:, :, 1, :, :7], x[:, :, 0, :, 5:], x[:, :, 1, :, 7:]], None),
    "different_types_of_rows": ((2, 3, 40), lambda x: [x[:, :, :8], x[:, :, 8:40].view(2, 3, 4, 8)[..., :5], x[:, :, 13]], None),
    "positions": ((2, 3, 2, 9, 8), lambda x: [x[:, :, 0], x[:, :, 1]], 4),
    "beams_first": ((3, 2, 2, 4, 9, 8), lambda x: [x.transpose(0, 1)[:, :, k, :, :5] for k in (0, 1)], None),
}


@pytest.mark.parametrize("name", list(PACKED))
def test_states_packed_into_one_buffer(name):
    import mpnn_amd
    from oracle import beam_oracle as orc

    shape, views, length = PACKED[name]
    buf = torch.randn(shape, generator=torch.Generator().manual_seed(3))
    parent = torch.tensor([[2, 0, 0], [1, 2, 1]])
    dev = buf.cuda()
    mpnn_amd.beam_reorder(views(dev), parent.cuda(), length)
    want = buf.clone()
    for x, y in zip(views(want), views(buf)):
        x.copy_(orc.reorder(y, parent, length))
    same = torch.equal(dev.cpu(), want)
    assert same


def test_states_that_share_a_byte_of_one_buffer_are_refused():
    import mpnn_amd

    x = torch.zeros(2, 3, 2, 4, 9, 8, device="cuda")
    parent = torch.zeros(2, 3, dtype=torch.int64, device="cuda")
    for pair in ([x[:, :, 0, :, :5], x[:, :, :, 3]], [x[:, :, 0, :, :5], x[:, :, 0, :, 4:]], [x[:, :, 0], x[:, :, 0, 1]],
                 [x[:, :, 1, :, :5], x[:, :, 1, :, :5]], [x[:, :, :, 0], x[:, :, 1, :, :2]]):
        with pytest.raises(ValueError, match="share memory"):
            mpnn_amd.beam_reorder(pair, parent)
