"""The lookup of an embedding table and the table's gradient against float64.

Tolerances.  A looked-up row is one product, rounded once: half a unit in the last place, and 2^-24 for the product in float32.  A row of the gradient is
a sum in float32 of at most n terms, added in some order: (n + 2) 2^-24 of the sum of magnitudes, and half a unit in the last place.
"""
import math

import pytest
import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -24}
SIZES = [(1, 1, 1), (1, 100, 192), (2, 1, 5), (5, 3, 1), (33, 100, 112), (64, 100, 192), (1000, 7, 33), (777, 5003, 204), (4096, 131, 8), (5000, 2, 40), (20000, 300, 24),
         (3, 70000, 16), (70000, 70001, 6), (4097, 1023, 260), (2049, 4096, 1032)]


def make(n, v, d, dtype, seed=0, offset=0):
    gen = torch.Generator(device="cuda").manual_seed(n + v + d + seed)
    ids = (torch.rand(n, generator=gen, device="cuda") ** 2 * v).long().clamp(max=v - 1)

    def one(rows):
        return torch.randn(rows * d + offset, generator=gen, device="cuda").to(dtype)[offset:].view(rows, d)

    return ids, one(v), one(n)


def reference(ids, weight, gy, scale, padding=None):
    """(value, allowed error) of the result and of the gradient."""
    half, tiny = HALF[weight.dtype], TINY[weight.dtype]
    y = scale * weight.double()[ids]
    live = torch.ones_like(ids, dtype=torch.bool) if padding is None else ids != padding
    g = gy.double().reshape(-1, gy.size(-1))[live.view(-1)] * scale
    at = ids.view(-1)[live.view(-1)]
    gw = torch.zeros(weight.shape, dtype=torch.float64, device=gy.device).index_add_(0, at, g)
    size = torch.zeros_like(gw).index_add_(0, at, g.abs())
    count = torch.bincount(at, minlength=weight.size(0))[:, None]
    off = (count + 2) * 2.0 ** -24 * size
    return (y, 2.0 ** -23 * y.abs() + half * y.abs() + tiny), (gw, off + half * (gw.abs() + off) + tiny)


def near(got, want):
    value, allowed = want
    assert got.shape == value.shape
    off = (got.double() - value).abs()
    assert (off <= allowed).all(), (off - allowed).max().item()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("n,v,d", SIZES)
def test_against_float64(n, v, d, offset, dtype):
    import gelib_b200 as G
    ids, weight, gy = make(n, v, d, dtype, offset=offset)
    weight.requires_grad_()
    scale = math.sqrt(d)
    for numbers in (ids, ids.int()):
        y = G.embedding(numbers, weight, scale)
        gw, = torch.autograd.grad(y, weight, gy)
        wants = reference(ids, weight.detach(), gy, scale)
        assert y.dtype == gw.dtype == dtype
        near(y.detach(), wants[0])
        near(gw, wants[1])


@pytest.mark.gpu
@pytest.mark.parametrize("n,v", [(100, 1), (3000, 5), (10, 3000), (5000, 3000), (300000, 90), (300000, 200000)])
def test_rows_met_often_and_never(n, v):
    """One row has half of the numbers, the last rows none; a repeated call gives the same bits."""
    import gelib_b200 as G
    ids, weight, gy = make(n, v, 20, torch.bfloat16)
    ids[torch.rand(n, device="cuda") < 0.5] = v // 2
    weight.requires_grad_()
    y = G.embedding(ids, weight)
    first, second = (torch.autograd.grad(y, weight, gy, retain_graph=True)[0] for _ in range(2))
    assert torch.equal(first, second)
    near(first, reference(ids, weight.detach(), gy, 1.0)[1])
    met = torch.zeros(v, dtype=torch.bool, device="cuda")
    met[ids] = True
    assert (first[~met] == 0).all()


@pytest.mark.gpu
def test_sorted_equal_and_descending_numbers():
    import gelib_b200 as G
    for n, v in ((5000, 700), (40000, 700)):
        _, weight, gy = make(n, v, 16, torch.float32)
        weight.requires_grad_()
        up = torch.arange(n, device="cuda") * v // n
        for ids in (up, up.flip(0), torch.full_like(up, v - 1), torch.zeros_like(up), up * 0 + (torch.arange(n, device="cuda") % 2) * (v - 1)):
            gw, = torch.autograd.grad(G.embedding(ids, weight), weight, gy)
            near(gw, reference(ids, weight.detach(), gy, 1.0)[1])


@pytest.mark.gpu
@pytest.mark.parametrize("padding", [0, 5, -1])
def test_a_row_for_padding_has_no_gradient(padding):
    import gelib_b200 as G
    for n, v in ((300, 12), (6000, 12), (40000, 5000)):
        ids, weight, gy = make(n, v, 24, torch.float32)
        ids[::3] = padding % v
        gy[::3] = float("nan")   # whatever comes from there
        weight.requires_grad_()
        gw, = torch.autograd.grad(G.embedding(ids, weight, 2.0, padding_idx=padding), weight, gy)
        near(gw, reference(ids, weight.detach(), gy, 2.0, padding % v)[1])
        assert (gw[padding] == 0).all()


@pytest.mark.gpu
def test_numbers_that_name_no_row():
    """NaN comes out, nothing goes back, and no memory but the table's is touched."""
    import gelib_b200 as G
    for n in (50, 5000, 40000):
        ids, weight, gy = make(n, 40, 24, torch.float32)
        bad = torch.zeros(n, dtype=torch.bool, device="cuda")
        bad[::7] = True
        odd = torch.tensor([-1, 40, 2 ** 31, -2 ** 31, 2 ** 62, -2 ** 63 + 1, 2 ** 32 + 1, 41], device="cuda")
        ids[bad] = odd[torch.arange(int(bad.sum()), device="cuda") % len(odd)]
        gy[bad] = float("nan")
        weight.requires_grad_()
        y = G.embedding(ids, weight)
        assert y[bad].isnan().all() and torch.equal(y[~bad], weight[ids[~bad]])
        gw, = torch.autograd.grad(y, weight, gy)
        near(gw, reference(ids[~bad], weight.detach(), gy[~bad], 1.0)[1])


@pytest.mark.gpu
def test_infinities_and_nan_stay_in_their_rows():
    import gelib_b200 as G
    for n in (500, 30000):
        ids, weight, gy = make(n, 50, 24, torch.float16)
        ids[3], ids[4] = 7, 9
        weight.requires_grad_()
        y = G.embedding(ids, weight)
        clean, = torch.autograd.grad(y, weight, gy, retain_graph=True)
        gy[3, 5], gy[4, 6] = float("nan"), float("inf")
        got, = torch.autograd.grad(y, weight, gy)
        assert got[7, 5].isnan() and got[9, 6] == float("inf")
        same = torch.ones_like(got, dtype=torch.bool)
        same[7, 5] = same[9, 6] = False
        assert torch.equal(got[same], clean[same])


@pytest.mark.gpu
def test_shapes_strides_streams_and_complex_rows():
    import gelib_b200 as G
    ids, weight, gy = make(60, 30, 24, torch.float32)
    want = G.embedding(ids, weight, 3.0)
    assert torch.equal(G.embedding(ids.view(3, 4, 5), weight, 3.0), want.view(3, 4, 5, 24))
    assert torch.equal(G.embedding(ids[7], weight, 3.0), want[7])
    assert torch.equal(G.embedding(torch.stack([ids, ids], 1)[:, 0], weight, 3.0), want)
    assert torch.equal(G.embedding(ids, weight.t().contiguous().t(), 3.0), want)
    wide = torch.zeros(30, 31, device="cuda")
    wide[:, 3:27] = weight
    assert torch.equal(G.embedding(ids, wide[:, 3:27], 3.0), want)
    assert torch.equal(G.embedding(ids, weight[:1].expand(30, 24), 3.0), 3.0 * weight[:1].expand(60, 24))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = G.embedding(ids, weight, 3.0)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(other, want)
    table = torch.view_as_complex(weight.reshape(30, 12, 2)).clone().requires_grad_()
    y = G.embedding(ids, table, 3.0)
    assert y.shape == (60, 12) and torch.equal(torch.view_as_real(y.detach()).reshape(60, 24), want)
    g, = torch.autograd.grad(y, table, torch.view_as_complex(gy.reshape(60, 12, 2)))
    near(torch.view_as_real(g).reshape(30, 24), reference(ids, weight, gy, 3.0)[1])
    leaf = weight.clone().requires_grad_()
    one, = torch.autograd.grad(G.embedding(ids, leaf), leaf, gy[:1].expand(60, 24))   # a gradient that is broadcast
    near(one, reference(ids, weight, gy[:1].expand(60, 24), 1.0)[1])


@pytest.mark.gpu
def test_sizes_of_nothing():
    import gelib_b200 as G
    for n, v, d in ((0, 5, 4), (0, 0, 4), (3, 5, 0), (0, 5, 0)):
        weight = torch.ones(v, d, device="cuda", requires_grad=True)
        y = G.embedding(torch.zeros(n, dtype=torch.long, device="cuda"), weight)
        assert y.shape == (n, d)
        gw, = torch.autograd.grad(y, weight, torch.ones_like(y))
        assert gw.shape == (v, d) and (gw == 0).all()


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """More than 2^31 elements of the table, and of the result."""
    import gelib_b200 as G
    if torch.cuda.get_device_properties(0).total_memory < 60 * 2 ** 30:
        pytest.skip("needs 60 GB of device memory")
    v, d = 1 << 20, 2056
    weight = torch.empty(v, d, dtype=torch.bfloat16, device="cuda").normal_().requires_grad_()
    ids = torch.arange(v - 1, -1, -1, device="cuda")
    y = G.embedding(ids, weight)
    at = torch.tensor([0, 1, v // 2, v - 1], device="cuda")
    assert torch.equal(y[at], weight[ids[at]])
    gw, = torch.autograd.grad(y, weight, y.detach())
    assert torch.equal(gw[at], weight[at])


@pytest.mark.gpu
def test_several_gradients_of_one_call_and_numbers_that_change_after_it():
    """The numbers are those of the forward call; its gradients can be had again, on two streams at a time."""
    import gelib_b200 as G
    for n, v in ((5000, 40), (90000, 300)):
        ids, weight, gy = make(n, v, 48, torch.float32)
        weight.requires_grad_()
        want = reference(ids, weight.detach(), gy, 1.0)[1]
        y = G.embedding(ids, weight)
        ids.zero_()
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        got = []
        for turn in range(6):
            with torch.cuda.stream(streams[turn % 2]):
                got.append(torch.autograd.grad(y, weight, gy, retain_graph=True)[0])
        torch.cuda.synchronize()
        near(got[0], want)
        assert all(torch.equal(g, got[0]) for g in got)


@pytest.mark.gpu
def test_two_captured_graphs_and_eager_calls_in_between():
    """Both graphs replay after either has changed its inputs; nothing in them waits for the host."""
    import gelib_b200 as G
    graphs = []
    for seed, (n, v) in enumerate(((3000, 50), (30000, 4000))):
        ids, weight, gy = make(n, v, 32, torch.float32, seed)
        weight.requires_grad_()

        def step(ids=ids, weight=weight, gy=gy):
            y = G.embedding(ids, weight, 2.0)
            return y.detach(), torch.autograd.grad(y, weight, gy)[0]

        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step()
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out, ids, weight, gy))
    for turn in range(2):
        for graph, out, ids, weight, gy in graphs:
            ids.copy_(ids.flip(0) if turn else ids)
            gy.mul_(1.5)
            G.embedding(ids[:40], weight)
            graph.replay()
        for graph, out, ids, weight, gy in graphs:
            wants = reference(ids, weight.detach(), gy, 2.0)
            near(out[0], wants[0])
            near(out[1], wants[1])


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_derivatives_that_do_not_exist_are_refused(native, monkeypatch):
    import torch.autograd.forward_ad as forward_ad
    import gelib_b200 as G
    if not native:
        monkeypatch.setattr(G._lib, "_native", G._lib._Declines())
    ids, weight, gy = make(6, 5, 4, torch.float32)
    leaf = weight.clone().requires_grad_()
    gy.requires_grad_()
    gw, = torch.autograd.grad(G.embedding(ids, leaf), leaf, gy, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        gw.sum().backward()
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="jvp|forward"):
            G.embedding(ids, forward_ad.make_dual(weight, torch.ones_like(weight)))


@pytest.mark.gpu
def test_the_python_host_side_gives_the_same(monkeypatch):
    import gelib_b200 as G
    ids, weight, gy = make(700, 90, 36, torch.bfloat16)
    weight.requires_grad_()

    def both():
        y = G.embedding(ids, weight, 1.5, padding_idx=-3)
        return y.detach(), torch.autograd.grad(y, weight, gy)[0]

    want = both()
    monkeypatch.setattr(G._lib, "_native", G._lib._Declines())
    assert all(torch.equal(a, b) for a, b in zip(both(), want))


@pytest.mark.gpu
def test_module():
    import gelib_b200 as G
    layer = G.Embedding(12, 8, scale=2.0, padding_idx=3, device="cuda")
    assert (layer.weight[3] == 0).all()
    ids = torch.tensor([[1, 3], [3, 11]], device="cuda")
    y = layer(ids)
    assert torch.equal(y, 2 * layer.weight[ids])
    y.sum().backward()
    assert layer.weight.grad[3].abs().sum() == 0 and (layer.weight.grad[1] == 2).all() and (layer.weight.grad[0] == 0).all()


def test_cpu_tensors_are_refused(cabi):
    import gelib_b200 as G
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        G.embedding(torch.zeros(2, dtype=torch.long), torch.zeros(5, 4))


REFUSALS = {
    "type of ids": ("ids must be an int64 or int32", dict(ids=torch.zeros(2))),
    "ids elsewhere": ("ids must be on the device of weight", dict(ids=torch.zeros(2, dtype=torch.long))),
    "no tensor": ("ids must be an int64 or int32", dict(ids=[1, 2])),
    "dimensions": ("2 dimensions", dict(weight=torch.zeros(5))),
    "double": ("float32, bfloat16 or float16", dict(weight=torch.zeros(5, 4, dtype=torch.float64))),
    "padding": ("padding_idx 5 is none of the 5 rows", dict(padding_idx=5)),
    "padding below": ("padding_idx -6 is none of the 5 rows", dict(padding_idx=-6)),
}


@pytest.mark.gpu
@pytest.mark.parametrize("which", list(REFUSALS))
def test_refusals(which):
    import gelib_b200 as G
    message, change = REFUSALS[which]
    args = dict(ids=torch.zeros(2, dtype=torch.long, device="cuda"), weight=torch.zeros(5, 4, device="cuda"))
    args.update({k: v.cuda() if isinstance(v, torch.Tensor) and which != "ids elsewhere" else v for k, v in change.items()})
    with pytest.raises(RuntimeError, match=message):
        G.embedding(**args)


C_REFUSALS = {
    "negative size": dict(n=-1),
    "2^30": dict(n=2 ** 31),
    "2^20": dict(d=2 ** 20 + 1, ldw=2 ** 21),
    "unknown type": dict(type=3),
    "8 or 4 bytes": dict(index_bytes=2),
    "null pointer": dict(y=0),
    "rows overlap": dict(ldw=7),
    "not aligned": dict(weight=4098),
    "state is not": dict(state=4100),
}


@pytest.mark.parametrize("message", list(C_REFUSALS))
def test_arguments_of_the_c_abi(cabi, message):
    """No kernel is launched: the addresses stand for nothing."""
    a = dict(y=4096, ids=4096, weight=4096, n=2, v=5, d=8, ldw=8, scale=1.0, padding=-1, index_bytes=8, type=0, state=4096)
    a.update(C_REFUSALS[message])
    assert cabi.gelib_embedding(*a.values(), None) == 2 and message in cabi.gelib_last_error().decode()


@pytest.mark.parametrize("message,change", [("negative size", dict(v=-1)), ("null pointer", dict(gy=0)), ("null pointer", dict(state=0)), ("not aligned", dict(gw=4098)),
                                            ("not 256-byte", dict(space=4100)), ("not 256-byte", dict(state=4100)), ("no workspace", dict(space=0))])
def test_arguments_of_the_c_abi_backward(cabi, message, change):
    a = dict(gw=4096, gy=4096, state=4096, n=2, v=5, d=8, scale=1.0, type=0, space=4096)
    a.update(change)
    assert cabi.gelib_embedding_back(*a.values(), None) == 2 and message in cabi.gelib_last_error().decode()


def test_state_and_workspace(cabi):
    """Numbers in order, twice, and blocks' counts of digits; at most two rows of partial sums for every 16 numbers."""
    for n, v, d, kind in ((1, 1, 1, 0), (64, 100, 192, 0), (65536, 100, 112, 0), (65537, 100, 112, 0), (32768, 65536, 2048, 1), (1 << 20, 262144, 128, 2)):
        assert 16 * n <= cabi.gelib_embedding_state_bytes(n, v) <= 16 * n + (1 << 20)
        assert 0 < cabi.gelib_embedding_workspace(n, v, d, kind) <= 8 * (d + 1) * (n // 16 + 1) + 1024
    assert cabi.gelib_embedding_workspace(0, 5, 4, 0) == 0 and cabi.gelib_embedding_workspace(5, 5, 4, 9) == 0 and cabi.gelib_embedding_state_bytes(0, 5) == 0
