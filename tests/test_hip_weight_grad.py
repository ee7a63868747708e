"""Weight and bias gradients from 8-bit checkpoints against the formula in 64 bits, at the values that are held.

Tolerance, with u = 2^-24: dy s is rounded once (u) and held in three bf16 terms (off by 2^-27 of itself at most) for
fp32, in two (2^-18) for the 16-bit types; the products with the integers are exact in fp32; a sum of M products in
fp32, in whatever order, is off by at most (M + 64) u of the sum of absolute values (64: the slabs and the terms);
the result is rounded once to its type: to an infinity from half a step beyond the type's largest number on (65520 in
fp16, whose sums of large products get there)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
U = 2.0 ** -24


def make(M, N, K, t, seed=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=gen) * torch.exp(torch.randn(M, 1, generator=gen))
    return torch.randn(M, N, generator=gen).to(TYPES[t]).cuda(), x.to(TYPES[t]).cuda()


def compare(dy, packed, t, got=None):
    from tango_amd.checkpoint import weight_grad
    dw, db = weight_grad(dy, packed, want_bias=True) if got is None else got
    assert dw.dtype == db.dtype == TYPES[t]
    spread = packed.scale.cpu().double().repeat_interleave(packed.group, 1)[:, :packed.values.size(1)]
    x = packed.values.cpu().double() * spread
    d = dy.detach().cpu().double().reshape(x.size(0), -1)
    M = x.size(0)
    info = torch.finfo(TYPES[t])
    split = 2.0 ** -27 if t == "fp32" else 2.0 ** -18
    for name, g, want, size, extra in (("dw", dw, d.t() @ x, d.abs().t() @ x.abs(), split + 2 * U), ("db", db, d.sum(0), d.abs().sum(0), 0.0)):
        g = g.detach().cpu().double()
        bound = ((M + 64) * U + extra) * size
        bound = bound + info.eps / 2 * (want.abs() + bound) + info.smallest_normal * info.eps
        assert g.shape == want.shape
        # a sum that may lie past half a step beyond the largest number may have become an infinity of its sign
        past = torch.isinf(g) & (want.abs() + bound >= info.max * (1 + info.eps / 4)) & (g.sign() == want.sign())
        assert (torch.isfinite(g) | past).all()
        over = float((torch.where(past, want, g) - want).abs().sub(bound).max()) if g.numel() else -1.0
        assert over <= 0, "%s: beyond its bound by %.3g" % (name, over)
    return dw, db


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("M,N,K,group", [
    (1, 1, 1, None), (1, 5, 7, 3), (2, 16, 16, 16), (31, 128, 128, None), (32, 128, 128, 128), (33, 129, 130, 128), (64, 41, 602, None),
    (100, 256, 500, 128), (129, 64, 257, 64), (257, 3, 130, 32), (1000, 200, 96, 24), (500, 17, 301, 43), (300, 300, 640, 256),
    (4000, 64, 64, 8), (40, 70, 33, 1), (10000, 40, 128, None), (5000, 256, 602, None),
])
def test_against_the_formula(M, N, K, group, t):
    from tango_amd.checkpoint import pack
    dy, x = make(M, N, K, t, seed=M + N)
    compare(dy, pack(x, group), t)


@pytest.mark.parametrize("t", sorted(TYPES))
def test_layouts(t):
    """Gradients with row strides, off alignment, transposed, broadcast, with leading dimensions."""
    from tango_amd.checkpoint import pack
    M, K = 210, 96
    base, x = make(M, 300, K, t, seed=3)
    p = pack(x, 32)
    for dy in (base[:, :128], base[:, 1:130], base[:, 3:4], base[:, ::2], base[:1].expand(M, 300), base[:, :1].expand(M, 64)):
        compare(dy, p, t)
    wide = pack(x.view(3, 70, K), 32)
    assert wide.shape == (3, 70, K)
    compare(base[:, :8].reshape(3, 70, 8), wide, t)


@pytest.mark.parametrize("t", sorted(TYPES))
def test_small_gradients_keep_their_precision(t):
    """Rows whose gradients differ by many powers of two, as after a mean over many rows."""
    from tango_amd.checkpoint import pack
    dy, x = make(600, 32, 64, t, seed=8)
    scale = torch.exp2(-torch.arange(600, device="cuda") % 12.0)[:, None]
    compare((dy * scale).to(TYPES[t]), pack(x, 64), t)
    compare((dy * 1e-6).to(TYPES[t]), pack(x, None), t)


def test_missing_values_stay_in_their_run():
    """A run that could not be held gives NaN in its own columns and nothing elsewhere; a gradient that is not finite
    reaches its own row."""
    from tango_amd.checkpoint import pack, weight_grad
    dy, x = make(100, 40, 64, "fp32", seed=4)
    x[17, 40] = float("inf")
    dw, db = weight_grad(dy, pack(x, 32), want_bias=True)
    assert torch.isnan(dw[:, 32:]).all() and torch.isfinite(dw[:, :32]).all() and torch.isfinite(db).all()
    dy, x = make(100, 40, 64, "fp32", seed=4)
    dy[3, 5] = float("inf")
    dw, db = weight_grad(dy, pack(x, 32), want_bias=True)
    assert not torch.isfinite(dw[5]).any() and torch.isinf(db[5])
    keep = torch.arange(40, device="cuda") != 5
    assert torch.isfinite(dw[keep]).all() and torch.isfinite(db[keep]).all()


def test_same_bits_every_time():
    from tango_amd.checkpoint import pack, weight_grad
    dy, x = make(30_000, 130, 200, "bf16", seed=9)
    p = pack(x, 64)
    first = weight_grad(dy, p, True)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, weight_grad(dy, p, True)))
    assert torch.equal(first[0], weight_grad(dy, p))


def test_captured_and_replayed():
    """A checkpoint and its weight gradient in one HIP graph, replayed over new inputs with eager work in between."""
    from tango_amd.checkpoint import pack, weight_grad
    dy, x = make(3000, 40, 96, "fp32", seed=2)
    weight_grad(dy, pack(x, 32), True)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        dw, db = weight_grad(dy, pack(x, 32), True)
    for seed in range(3):
        for a, b in zip((dy, x), make(3000, 40, 96, "fp32", seed=10 + seed)):
            a.copy_(b)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((dw, db), weight_grad(dy, pack(x, 32), True)))


def test_two_streams_at_once():
    from tango_amd.checkpoint import pack, weight_grad
    cases = [make(20_000, 64, 130, t, seed=s) for s, t in ((1, "fp32"), (2, "bf16"))]
    packed = [pack(x, 64) for _, x in cases]
    want = [weight_grad(dy, p, True) for (dy, _), p in zip(cases, packed)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(4):
        got = []
        for s, (dy, _), p in zip(streams, cases, packed):
            with torch.cuda.stream(s):
                got.append(weight_grad(dy, p, True))
        torch.cuda.synchronize()
        assert all(torch.equal(u, w) for a, b in zip(want, got) for u, w in zip(a, b))


def test_offsets_beyond_32_bits():
    """Rows whose elements lie past 2^31 in both operands: zeros but for the first and the last rows."""
    from tango_amd.checkpoint import pack, weight_grad
    M, N, K = 8_500_000, 256, 256
    assert M * N > 1 << 31
    dy, x = torch.zeros(M, N, dtype=torch.bfloat16, device="cuda"), torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    a, b = make(400, N, K, "bf16", seed=6)
    for whole, part in ((dy, a), (x, b)):
        whole[:200], whole[-200:] = part[:200], part[200:]
    p, q = pack(x, 64), pack(b, 64)
    del x
    assert torch.equal(p.values[-200:], q.values[200:]) and torch.equal(p.scale[-200:], q.scale[200:])
    compare(a, q, "bf16", weight_grad(dy, p, True))


def test_no_rows_and_no_columns():
    from tango_amd.checkpoint import pack, weight_grad
    z = lambda *s: torch.zeros(*s, device="cuda")
    for M, N, K in ((0, 3, 4), (5, 3, 0), (5, 0, 4), (0, 0, 0)):
        dw, db = weight_grad(z(M, N) + 1, pack(z(M, K)), True)
        assert dw.shape == (N, K) and db.shape == (N,) and (dw == 0).all() and (db == M).all()


def test_linear_layer():
    """The layer's output is torch's linear layer; its gradients are the formula's at the held input."""
    from tango_amd.checkpoint import CheckpointLinear, pack
    torch.manual_seed(3)
    layer = CheckpointLinear(96, 40, group=32).cuda()
    plain = torch.nn.Linear(96, 40).cuda()
    plain.load_state_dict(layer.state_dict())
    x = torch.randn(7, 50, 96, device="cuda", requires_grad=True)
    dy = torch.randn(7, 50, 40, device="cuda")
    y, z = layer(x), plain(x)
    assert torch.equal(y, z)
    dx, dw, db = torch.autograd.grad(y, (x, layer.weight, layer.bias), dy)
    assert torch.equal(dx, torch.autograd.grad(z, x, dy)[0])
    compare(dy, pack(x, 32), "fp32", (dw, db))
    # what is not asked for is not computed, and a layer without a bias has none
    layer.weight.requires_grad_(False)
    y = layer(x)
    assert y.grad_fn.held is None
    dx2, db2 = torch.autograd.grad(y, (x, layer.bias), dy)
    assert torch.equal(dx2, dx) and torch.allclose(db2, db, rtol=1e-5, atol=1e-5)
    bare = CheckpointLinear(96, 40, bias=False).cuda()
    torch.autograd.grad(bare(x.detach()).sum(), bare.weight)


@pytest.mark.parametrize("t", ["bf16", "fp16"])
def test_linear_layer_under_autocast(t):
    """Autocast runs the layer in its type on fp32 parameters; the gradients reach the parameters in theirs."""
    from tango_amd.checkpoint import CheckpointLinear, pack
    torch.manual_seed(4)
    layer, plain = CheckpointLinear(96, 40, group=32).cuda(), torch.nn.Linear(96, 40).cuda()
    plain.load_state_dict(layer.state_dict())
    for x in (torch.randn(50, 96, device="cuda"), torch.randn(50, 96, device="cuda", dtype=TYPES[t])):
        x.requires_grad_()
        dy = torch.randn(50, 40, device="cuda", dtype=TYPES[t])
        with torch.autocast("cuda", TYPES[t]):
            y, z = layer(x), plain(x)
        assert y.dtype == TYPES[t] and torch.equal(y, z)
        dx, dw, db = torch.autograd.grad(y, (x, layer.weight, layer.bias), dy)
        assert torch.equal(dx, torch.autograd.grad(z, x, dy)[0]) and dx.dtype == x.dtype
        assert dw.dtype == db.dtype == torch.float32
        compare(dy, pack(x.to(TYPES[t]), 32), t, (dw.to(TYPES[t]), db.to(TYPES[t])))


def test_held_input_is_released_by_the_backward_pass():
    """As what torch saves is: an output that lives on keeps nothing, and a second backward pass is refused."""
    from tango_amd.checkpoint import CheckpointLinear
    layer = CheckpointLinear(512, 8).cuda()
    x = torch.randn(4096, 512, device="cuda")
    before = torch.cuda.memory_allocated()
    y = layer(x)
    kept = torch.cuda.memory_allocated() - before
    loss = y.sum()
    loss.backward()
    small = 4 * (y.numel() + 512 * 8 + 8) + 16384  # y and the gradients, and rounding up
    assert kept > x.numel() and torch.cuda.memory_allocated() - before < small < x.numel()
    with pytest.raises(RuntimeError, match="second time"):
        loss.backward()


def test_refusals():
    from tango_amd.checkpoint import CheckpointLinear, checkpoint_linear, pack, weight_grad
    dy, x = make(10, 8, 16, "fp32")
    p = pack(x)
    for bad in (dy[:9], dy.double(), dy.cpu(), dy.view(2, 5, 8)[:1]):
        with pytest.raises(RuntimeError):
            weight_grad(bad, p)
    with pytest.raises(TypeError):
        weight_grad(dy, x)
    with pytest.raises(RuntimeError):
        checkpoint_linear.apply(x, torch.zeros(4, 16, device="cuda", dtype=torch.bfloat16), None)
    with pytest.raises(ValueError):
        CheckpointLinear(4, 4, group=0)
