"""The attention over a graph's edges and its gradient against the formulas in 64 bits on the CPU.

Tolerances.  With u = 2^-24 and absolute values throughout: a logit is a dot product of dim terms in fp32 times a
rounded factor, off by at most a = (dim + 8) u scale sum|q||k| plus, from the subtraction of the maximum and from the
stored denominator, 4 u (max|logit| + log2(edges)); the hardware's 2^x adds 4 u.  A weight is then off by the factor
w = 2 a + 16 u (a in natural units, twice for numerator and denominator).  Sums of n terms add n u of the sum of
absolute terms.  So an output is off by at most (w + (n + dim + 16) u) sum p|v| and half a step of its type, and a gradient
by (2 w + (2 n + 2 dim + 64) u) times the formula with every difference and product taken in absolute values: the same
sums, run on |q|, |k|, |v|, |dout|.  The hardware's 2^x gives 0 where the result is below fp32's smallest normal number
2^-126, so a weight may be off by that much absolutely: n 2^-126 times the largest factor a weight meets in the sum."""
import math

import numpy as np
import pytest
import torch

from gpu_util import powerlaw_graph

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
U = 2.0 ** -24


def make_graph(src, dst, num_src, num_dst):
    from tango_amd.graph import Graph
    from tango_amd.util import graph_preprocess
    return graph_preprocess(Graph(torch.as_tensor(src).cuda(), torch.as_tensor(dst).cuda(), num_src, num_dst))


def half_step(t, x):
    """Half a step of type t at |x|, and of its smallest numbers."""
    info = torch.finfo(t)
    return info.eps / 2 * x.abs() + info.smallest_normal * info.eps


def formulas(src, dst, q, k, v, dout, scale, mask):
    """Outputs, gradients and the bounds above; everything float64 on the CPU."""
    src, dst = torch.as_tensor(src).cpu(), torch.as_tensor(dst).cpu()
    if mask is not None:
        src, dst = src[mask.cpu()], dst[mask.cpu()]
    q, k, v, dout = (t.detach().cpu().double() for t in (q, k, v, dout))
    n, H, D = q.shape
    rep = H // k.size(1)
    ke, ve = k[src].repeat_interleave(rep, 1), v[src].repeat_interleave(rep, 1)
    qe, oe = q[dst], dout[dst]
    to_dst = lambda e: torch.zeros((n,) + e.shape[1:], dtype=torch.float64).index_add_(0, dst, e)
    to_src = lambda e: torch.zeros(k.shape, dtype=torch.float64).index_add_(0, src, e.view(-1, H // rep, rep, D).sum(2))
    logit = (qe * ke).sum(2) * scale
    top = torch.full((n, H), -math.inf, dtype=torch.float64).scatter_reduce(0, dst[:, None].expand(-1, H), logit, "amax")
    p = torch.exp(logit - top[dst])
    p = p / to_dst(p)[dst]
    out = to_dst(p[:, :, None] * ve)
    dp = (oe * ve).sum(2)
    delta = to_dst(p * dp)
    ds = p * (dp - delta[dst]) * scale
    want = [out, to_dst(ds[:, :, None] * ke), to_src(ds[:, :, None] * qe), to_src(p[:, :, None] * oe)]
    # bounds
    edges = int(max(torch.bincount(dst, minlength=1).max(), torch.bincount(src, minlength=1).max() * rep)) if len(src) else 0
    size = float(((qe.abs() * ke.abs()).sum(2) * abs(scale)).max()) if len(src) else 0.0
    a = (D + 8) * U * size + 4 * U * (size + math.log2(edges + 2))
    w = 2 * a + 16 * U
    adp = (oe.abs() * ve.abs()).sum(2)
    ads = (p * (adp + to_dst(p * adp)[dst]) * abs(scale))[:, :, None]
    fwd, bwd = w + (edges + D + 16) * U, 2 * w + (2 * edges + 2 * D + 64) * U
    bound = [fwd * to_dst(p[:, :, None] * ve.abs()), bwd * to_dst(ads * ke.abs()), bwd * to_src(ads * qe.abs()),
             bwd * to_src(p[:, :, None] * oe.abs())]
    if len(src):
        most = lambda e: float(e.abs().max())
        lost, factor = edges * 2.0 ** -126, 2 * most(adp) * abs(scale)
        for b, largest in zip(bound, (most(ve), factor * most(ke), factor * most(qe), most(oe))):
            b += lost * largest
    return want, bound


def check(got, want, bound, t):
    for name, g, x, b in zip(("out", "dq", "dk", "dv"), got, want, bound):
        g = g.detach().cpu().double()
        assert g.shape == x.shape and torch.isfinite(g).all(), name
        over = ((g - x).abs() - b - half_step(t, x) - half_step(t, b)).max() if g.numel() else torch.tensor(-1.0)
        assert over <= 0, "%s: beyond its bound by %.3g" % (name, over)


def inputs(num_src, num_dst, heads, kv, dim, t, seed=0, peak=1.0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)
    q, k, v, dout = peak * r(num_dst, heads, dim), r(num_src, kv, dim), r(num_src, kv, dim), r(num_dst, heads, dim)
    return [x.to(t).cuda() for x in (q, k, v, dout)]


def run(graph, q, k, v, dout, **kw):
    from tango_amd.graph_attention import graph_attention
    leaves = [x.detach().clone().requires_grad_() for x in (q, k, v)]
    out = graph_attention(graph, *leaves, **kw)
    return [out, *torch.autograd.grad(out, leaves, dout)]


@pytest.mark.parametrize("cap", [1, 3, 16, 64, 512])
@pytest.mark.parametrize("rows", [1, 10, 255, 256, 257, 5000])
def test_items_cover_every_edge_once(rows, cap):
    """The cut into items: every slot once, rows in slot order, no item longer than the cap, longest first, empty rows
    present, parts of a row consecutive."""
    from tango_amd.graph_attention import AttentionItems
    gen = torch.Generator().manual_seed(rows + cap)
    degree = (torch.rand(rows, generator=gen) ** 6 * 2000).long()
    degree[:10] = torch.tensor([0, 1, 200, 0, 64, 65, 3, 0, 129, 2])[:rows]
    indptr = torch.zeros(rows + 1, dtype=torch.int64)
    indptr[1:] = torch.cumsum(degree, 0)
    a = AttentionItems(indptr.cuda(), torch.zeros(int(indptr[-1]), dtype=torch.int32, device="cuda"), None, cap=cap)
    items, split = a.items.cpu().long(), a.split.cpu().long()
    lengths = items[:, 2] - items[:, 1]
    assert (lengths[:-1] >= lengths[1:]).all() and int(lengths.max()) <= cap and int(lengths.min()) >= 0
    pieces = torch.clamp((degree + cap - 1) // cap, min=1)
    assert torch.equal(torch.bincount(items[:, 0], minlength=rows), pieces)
    order = torch.argsort(items[:, 0] * (int(indptr[-1]) + 1) + items[:, 1], stable=True)
    items = items[order]
    starts = torch.cumsum(pieces, 0) - pieces
    assert torch.equal(items[starts, 1], indptr[:-1]) and torch.equal(items[starts + pieces - 1, 2], indptr[1:])
    inner = torch.ones(len(items), dtype=torch.bool)
    inner[starts] = False
    assert torch.equal(items[1:, 1][inner[1:]], items[:-1, 2][inner[1:]])
    cut = torch.nonzero(pieces > 1).flatten()
    assert sorted(split[:, 0].tolist()) == cut.tolist() and a.struct.num_parts == int(pieces[cut].sum())
    parts = torch.full((rows,), -1)
    parts[split[:, 0]] = split[:, 1]
    assert torch.equal(split[:, 2] - split[:, 1], pieces[split[:, 0]])
    nth = torch.arange(len(items)) - starts[items[:, 0]]
    assert torch.equal(items[:, 3], torch.where(pieces[items[:, 0]] > 1, parts[items[:, 0]] + nth, -1))
    taken = torch.sort(items[items[:, 3] >= 0, 3]).values
    assert torch.equal(taken, torch.arange(a.struct.num_parts))


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("dim", [1, 2, 3, 4, 7, 8, 12, 16, 24, 31, 32, 40, 64, 72, 100, 128, 136, 250, 256])
def test_dims(dim, t):
    rng = np.random.default_rng(dim)
    src, dst = powerlaw_graph(rng, 60, 700)
    g = make_graph(src, dst, 60, 60)
    x = inputs(60, 60, 3, 3, dim, TYPES[t], seed=dim)
    scale = 1.0 / math.sqrt(dim)
    check(run(g, *x), *formulas(src, dst, *x, scale, None), TYPES[t])


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("heads,kv", [(1, 1), (2, 1), (4, 4), (8, 2), (5, 5), (6, 3), (16, 16), (12, 1), (9, 9)])
@pytest.mark.parametrize("dim", [4, 32, 41])
def test_head_layouts(heads, kv, dim, t):
    rng = np.random.default_rng(heads * 100 + kv)
    src, dst = rng.integers(0, 50, 400), rng.integers(0, 33, 400)
    g = make_graph(src, dst, 50, 33)
    x = inputs(50, 33, heads, kv, dim, TYPES[t], seed=heads)
    check(run(g, *x, scale=0.3), *formulas(src, dst, *x, 0.3, None), TYPES[t])


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("edges", [1, 2, 3, 4, 5, 63, 64, 65, 127, 128, 129, 1000, 20000])
def test_row_lengths(edges, t):
    """One destination with that many in-edges among short and empty rows; one source with that many out-edges."""
    rng = np.random.default_rng(edges)
    src = np.concatenate([rng.integers(0, 300, edges), np.full(edges, 7), [0, 1, 2]])
    dst = np.concatenate([np.full(edges, 5), rng.integers(6, 290, edges), [10, 11, 11]])
    g = make_graph(src, dst, 300, 300)
    x = inputs(300, 300, 2, 1, 32, TYPES[t], seed=edges)
    check(run(g, *x), *formulas(src, dst, *x, 1 / math.sqrt(32), None), TYPES[t])


@pytest.mark.parametrize("checkpoint", [None, "int8"])
@pytest.mark.parametrize("num_src,num_dst,edges", [(1, 1, 0), (1, 1, 1), (1, 1, 9), (5, 0, 0), (0, 5, 0), (0, 0, 0), (7, 3, 0), (1, 40, 40)])
def test_smallest_graphs(num_src, num_dst, edges, checkpoint):
    rng = np.random.default_rng(1)
    src = rng.integers(0, max(num_src, 1), edges)
    dst = rng.permutation(np.arange(edges) % max(num_dst, 1))
    g = make_graph(src.astype(np.int64), dst.astype(np.int64), num_src, num_dst)
    x = inputs(num_src, num_dst, 2, 2, 16, torch.float32, seed=3)
    got = run(g, *x, checkpoint=checkpoint)
    if checkpoint is None:
        check(got, *formulas(src.astype(np.int64), dst.astype(np.int64), *x, 0.25, None), torch.float32)
    for a, b in zip(got, (x[0], x[0], x[1], x[2])):
        assert a.shape == b.shape and torch.isfinite(a).all()
    if edges == 0:
        assert all((a == 0).all() for a in got)


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("dim", [16, 32, 33])
def test_masked_edges(dim, t):
    """Random masks, rows that a mask leaves empty, and whatever stands in masked places: infinities, NaN, the type's
    lowest value in the keys and values that only masked edges read."""
    rng = np.random.default_rng(11)
    n, m = 80, 3000
    src, dst = powerlaw_graph(rng, n, m)
    g = make_graph(src, dst, n, n)
    t = TYPES[t]
    x = inputs(n, n, 4, 2, dim, t, seed=4)
    keep = torch.from_numpy(rng.random(m) < 0.5)
    keep[torch.as_tensor(dst) == 0] = False      # the largest hub keeps nothing
    keep[torch.as_tensor(dst) == 17] = False
    for node in (1, 2, 5):                        # hubs as sources
        keep[torch.as_tensor(src) == node] = False
    clean = formulas(src, dst, *x, 0.2, keep)
    x[1][1], x[2][1] = float("nan"), float("inf")
    x[1][2], x[2][2] = -float("inf"), float("nan")
    x[1][5], x[2][5] = torch.finfo(t).min, torch.finfo(t).min
    got = run(g, *x, scale=0.2, edge_mask=keep.cuda())
    check(got, *clean, t)
    assert (got[0][0] == 0).all() and (got[1][0] == 0).all() and (got[2][1] == 0).all() and (got[3][2] == 0).all()
    none = run(g, *x, edge_mask=torch.zeros(m, dtype=torch.bool, device="cuda"))
    assert all((a == 0).all() for a in none)
    x = inputs(n, n, 4, 2, dim, t, seed=4)
    for a, b in zip(run(g, *x, edge_mask=torch.ones(m, dtype=torch.bool, device="cuda")), run(g, *x)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dim", [32, 5])
def test_lowest_logits_and_missing_values(dim):
    """Keys of the type's lowest value give logits of -inf or the lowest number: no weight beside an ordinary edge, and
    a row of nothing but -inf logits has no weight to give.  A NaN that takes part reaches its rows and no others."""
    n = 6
    src = torch.tensor([0, 1, 0, 1, 2, 0, 3, 0])
    dst = torch.tensor([0, 0, 1, 2, 3, 3, 4, 5])
    g = make_graph(src, dst, n, n)
    q, k, v, _ = inputs(n, n, 1, 1, dim, torch.float32, seed=9)
    q[:] = q.abs() + 0.5
    k[1] = torch.finfo(torch.float32).min
    k[3] = float("nan")
    from tango_amd.graph_attention import graph_attention
    out = graph_attention(g, q, k, v, scale=1.0)
    assert torch.equal(out[0], v[0]) and torch.equal(out[1], v[0]) and torch.equal(out[5], v[0])
    assert (out[2] == 0).all()  # -inf alone
    assert torch.isfinite(out[3]).all() and torch.isnan(out[4]).all()


def test_far_logits():
    """Logits of thousands: the maximum is subtracted before anything is raised to a power."""
    rng = np.random.default_rng(2)
    src, dst = powerlaw_graph(rng, 40, 900)
    g = make_graph(src, dst, 40, 40)
    x = inputs(40, 40, 2, 2, 64, torch.float32, seed=8, peak=40.0)
    check(run(g, *x, scale=1.0), *formulas(src, dst, *x, 1.0, None), torch.float32)
    check(run(g, *x, scale=-1.0), *formulas(src, dst, *x, -1.0, None), torch.float32)
    check(run(g, *x, scale=0.0), *formulas(src, dst, *x, 0.0, None), torch.float32)


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 32), (8, 2, 64), (3, 3, 41), (2, 2, 250)])
def test_from_checkpoints(heads, kv, dim, t):
    """With checkpoints the output is that of the call without, and the gradients are the attention's at the held
    values."""
    from tango_amd.checkpoint import pack, unpack
    rng = np.random.default_rng(dim)
    src, dst = powerlaw_graph(rng, 300, 6000)
    g = make_graph(src, dst, 300, 300)
    t = TYPES[t]
    x = inputs(300, 300, heads, kv, dim, t, seed=dim)
    mask = torch.from_numpy(rng.random(6000) < 0.8).cuda()
    held = [unpack(pack(a.flatten(1), dim), torch.float32).view_as(a) for a in x[:3]]
    want, bound = formulas(src, dst, *held, x[3], 0.2, mask)
    got = run(g, *x, scale=0.2, edge_mask=mask, checkpoint="int8")
    plain = run(g, *x, scale=0.2, edge_mask=mask)
    assert torch.equal(got[0], plain[0])
    check([want[0]] + got[1:], want, bound, t)


def test_gradient_against_differences():
    """Central differences of the 64-bit formula's loss sum(out * dout) along random directions, step 1e-5: their own
    error is some 1e-9 of the loss' third derivative and 1e-11 of its value."""
    rng = np.random.default_rng(6)
    src, dst = powerlaw_graph(rng, 30, 200)
    g = make_graph(src, dst, 30, 30)
    x = inputs(30, 30, 2, 1, 12, torch.float32, seed=6)
    got = run(g, *x, scale=0.4)
    _, bound = formulas(src, dst, *x, 0.4, None)
    loss = lambda *a: float((formulas(src, dst, *a, x[3], 0.4, None)[0][0] * x[3].cpu().double()).sum())
    base = [a.cpu().double() for a in x[:3]]
    gen = torch.Generator().manual_seed(1)
    for i in range(3):
        for _ in range(4):
            way = torch.randn(base[i].shape, generator=gen, dtype=torch.float64)
            up, down = list(base), list(base)
            up[i], down[i] = base[i] + 1e-5 * way, base[i] - 1e-5 * way
            slope = (loss(*up) - loss(*down)) / 2e-5
            mine = float((got[1 + i].cpu().double() * way).sum())
            room = float(((bound[1 + i] + half_step(torch.float32, got[1 + i].cpu().double())) * way.abs()).sum()) + 1e-5
            assert abs(mine - slope) <= room


@pytest.mark.parametrize("t", sorted(TYPES))
def test_strides(t):
    """Views of one fused projection, heads in another order, rows off alignment, a broadcast gradient."""
    from tango_amd.graph_attention import graph_attention
    rng = np.random.default_rng(3)
    n, H, D = 70, 4, 32
    src, dst = powerlaw_graph(rng, n, 900)
    g = make_graph(src, dst, n, n)
    t = TYPES[t]
    gen = torch.Generator().manual_seed(12)
    fused = torch.randn(n, 3 * H * D + 1, generator=gen).to(t).cuda()
    dout = torch.randn(n, H, D, generator=gen).to(t).cuda()
    views = [
        [fused[:, i * H * D:(i + 1) * H * D].view(n, H, D) for i in range(3)],
        [fused[:, 1 + i * H * D:1 + (i + 1) * H * D].view(n, H, D) for i in range(3)],
        [fused[:, :-1].view(n, H, 3, D)[:, :, i] for i in range(3)],
        [x.permute(1, 0, 2).contiguous().permute(1, 0, 2) for x in fused[:, :-1].view(n, 3, H, D).unbind(1)],
        [x.transpose(1, 2).contiguous().transpose(1, 2) for x in fused[:, :-1].view(n, 3, H, D).unbind(1)],
        [fused[:, :D].reshape(n, 1, D).expand(n, H, D), fused[:1, D:2 * D].reshape(1, 1, D).expand(n, H, D),
         fused[:, 2 * D:(2 + H) * D].view(n, H, D)],
    ]
    for q, k, v in views:
        want, bound = formulas(src, dst, q, k, v, dout, 0.25, None)
        for checkpoint in (None, "int8"):
            out = graph_attention(g, q, k, v, scale=0.25, checkpoint=checkpoint)
            check([out], want, bound, t)
        leaves = [a.detach().requires_grad_() for a in (q, k, v)]
        out = graph_attention(g, *leaves, scale=0.25)
        check([out, *torch.autograd.grad(out, leaves, dout)], want, bound, t)
    q, k, v = [a.detach().clone().requires_grad_() for a in views[0]]
    ones = torch.ones(1, 1, 1, device="cuda", dtype=t).expand(n, H, D)
    grads = torch.autograd.grad(graph_attention(g, q, k, v, scale=0.25), (q, k, v), ones)
    want, bound = formulas(src, dst, q, k, v, ones, 0.25, None)
    check([want[0], *grads], want, bound, t)


@pytest.mark.parametrize("checkpoint", [None, "int8"])
@pytest.mark.parametrize("layout", ["transposed", "broadcast", "sliced"])
def test_heads_of_one_column(layout, checkpoint):
    """Heads of one column whose heads lie apart, or on each other: held and attended as their contiguous copies are."""
    from tango_amd.graph_attention import graph_attention
    n, H = 50, 6
    gen = torch.Generator().manual_seed(8)
    make = {"transposed": lambda: torch.randn(H, n, 1, generator=gen).cuda().transpose(0, 1),
            "broadcast": lambda: torch.randn(n, 1, 1, generator=gen).cuda().expand(n, H, 1),
            "sliced": lambda: torch.randn(n, H, 3, generator=gen).cuda()[:, :, 1:2]}[layout]
    g = make_graph(torch.randint(0, n, (400,), generator=gen), torch.randint(0, n, (400,), generator=gen), n, n)
    results = []
    x = [make() for _ in range(3)]
    dout = torch.randn(n, H, 1, generator=gen).cuda()
    for leaves in ([t.detach().requires_grad_() for t in x], [t.contiguous().requires_grad_() for t in x]):
        out = graph_attention(g, *leaves, checkpoint=checkpoint)
        results.append([out.detach(), *torch.autograd.grad(out, leaves, dout)])
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_gradients_of_shared_and_broadcast_leaves():
    """One leaf for keys and values, one row of queries for every destination: autograd adds what belongs together."""
    from tango_amd.graph_attention import graph_attention
    rng = np.random.default_rng(13)
    src, dst = powerlaw_graph(rng, 50, 800)
    g = make_graph(src, dst, 50, 50)
    gen = torch.Generator().manual_seed(3)
    kv, q0 = torch.randn(50, 2, 24, generator=gen).cuda().requires_grad_(), torch.randn(1, 2, 24, generator=gen).cuda().requires_grad_()
    dout = torch.randn(50, 2, 24, generator=gen).cuda()
    out = graph_attention(g, q0.expand(50, 2, 24), kv, kv, scale=0.3)
    dq0, dkv = torch.autograd.grad(out, (q0, kv), dout)
    want, bound = formulas(src, dst, q0.expand(50, 2, 24), kv, kv, dout, 0.3, None)
    slack = 64 * U  # of the sums autograd makes
    for got, x, b in ((dq0, want[1].sum(0, keepdim=True), bound[1].sum(0, keepdim=True) + slack * want[1].abs().sum(0, keepdim=True)),
                      (dkv, want[2] + want[3], bound[2] + bound[3] + slack * (want[2].abs() + want[3].abs()))):
        assert ((got.cpu().double() - x).abs() <= b + 1e-30).all()


@pytest.mark.parametrize("which", [(0,), (1,), (2,), (0, 2), (1, 2)])
def test_only_some_inputs_need_gradients(which):
    from tango_amd.graph_attention import graph_attention
    rng = np.random.default_rng(21)
    src, dst = powerlaw_graph(rng, 90, 2500)
    g = make_graph(src, dst, 90, 90)
    x = inputs(90, 90, 2, 2, 16, torch.float32, seed=1)
    full = run(g, *x)
    leaves = [a.detach().clone().requires_grad_(i in which) for i, a in enumerate(x[:3])]
    for checkpoint in (None, "int8"):
        out = graph_attention(g, *leaves, checkpoint=checkpoint)
        grads = torch.autograd.grad(out, [leaves[i] for i in which], x[3])
        if checkpoint is None:
            for i, got in zip(which, grads):
                assert torch.equal(got, full[1 + i])
    assert not graph_attention(g, *x[:3]).requires_grad


@pytest.mark.parametrize("checkpoint", [None, "int8"])
@pytest.mark.parametrize("t,heads,kv", [("fp32", 8, 8), ("fp32", 8, 2), ("bf16", 20, 20)])
def test_rows_beyond_the_caches(t, heads, kv, checkpoint):
    """Tensors larger than the L2s together: the other order of workgroups, wider tiles."""
    from tango_amd.checkpoint import pack, unpack
    rng = np.random.default_rng(77)
    n, m, D = 22000, 40000, 32
    src, dst = powerlaw_graph(rng, n, m)
    g = make_graph(src, dst, n, n)
    x = inputs(n, n, heads, kv, D, TYPES[t], seed=7)
    got = run(g, *x, checkpoint=checkpoint)
    held = x[:3] if checkpoint is None else [unpack(pack(a.flatten(1), D), torch.float32).view_as(a) for a in x[:3]]
    want, bound = formulas(src, dst, *held, x[3], 1 / math.sqrt(D), None)
    if checkpoint:
        got[0], want[0], bound[0] = got[1], want[1], bound[1]  # the output is not that of the held values
    check(got, want, bound, TYPES[t])


def test_same_bits_every_time():
    """No result depends on the order in which workgroups run."""
    rng = np.random.default_rng(30)
    src, dst = powerlaw_graph(rng, 4000, 300_000)
    g = make_graph(src, dst, 4000, 4000)
    x = inputs(4000, 4000, 8, 4, 32, torch.bfloat16, seed=5)
    for checkpoint in (None, "int8"):
        first = run(g, *x, checkpoint=checkpoint)
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(first, run(g, *x, checkpoint=checkpoint)))


def test_edges_in_destination_order():
    """A graph whose slots are its edge ids walks masks without an indirection: same results."""
    from tango_amd.graph import Graph
    from tango_amd.util import graph_preprocess
    rng = np.random.default_rng(8)
    src, dst = powerlaw_graph(rng, 100, 3000)
    g = Graph(torch.as_tensor(src).cuda(), torch.as_tensor(dst).cuda(), 100)
    r = graph_preprocess(g.reorder_edges_by_dst())
    g = graph_preprocess(g)
    assert r.csc_slots_are_edge_ids and not g.csc_slots_are_edge_ids
    mask = torch.rand(3000, device="cuda") < 0.5
    x = inputs(100, 100, 2, 2, 16, torch.float32)
    for a, b in zip(run(g, *x, edge_mask=mask)[:2], run(r, *x, edge_mask=mask[r.edge_order])[:2]):
        assert torch.equal(a, b)
    check(run(r, *x, edge_mask=mask[r.edge_order]), *formulas(src, dst, *x, 0.25, mask), torch.float32)


def test_captured_forward():
    """The forward pass captures and replays (new inputs, eager work between the replays); the backward refuses, and so
    does a capture on a graph whose items have not been built."""
    from tango_amd.graph_attention import graph_attention, prepare_attention
    rng = np.random.default_rng(40)
    src, dst = powerlaw_graph(rng, 500, 30_000)
    q, k, v, _ = inputs(500, 500, 4, 4, 32, torch.float32)
    g = prepare_attention(make_graph(src, dst, 500, 500))
    graph_attention(g, q, k, v)
    torch.cuda.synchronize()
    graphs = []
    for scale in (0.1, 0.5):
        cg = torch.cuda.CUDAGraph()
        with torch.cuda.graph(cg):
            out = graph_attention(g, q, k, v, scale=scale)
        graphs.append((cg, out, scale))
    for seed in range(3):
        for a, b in zip((q, k, v), inputs(500, 500, 4, 4, 32, torch.float32, seed=50 + seed)):
            a.copy_(b)
        for cg, out, scale in graphs:
            cg.replay()
        torch.cuda.synchronize()
        for cg, out, scale in graphs:
            assert torch.equal(out, graph_attention(g, q, k, v, scale=scale))


def test_on_another_stream():
    """Forward and backward on a side stream, on a graph first used there."""
    rng = np.random.default_rng(41)
    src, dst = powerlaw_graph(rng, 800, 40_000)
    x = inputs(800, 800, 2, 2, 64, torch.float32)
    want = run(make_graph(src, dst, 800, 800), *x)
    g = make_graph(src, dst, 800, 800)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run(g, *x)
    here = run(g, *x)
    s.synchronize()
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, got, here))


def test_two_streams_at_once():
    """Calls on two streams in flight together, each with rows that leave parts in its scratch."""
    rng = np.random.default_rng(43)
    src, dst = powerlaw_graph(rng, 600, 60_000)
    g = make_graph(src, dst, 600, 600)
    cases = [(inputs(600, 600, 4, 2, 32, torch.float32, seed=s), kw) for s, kw in ((1, {}), (2, dict(checkpoint="int8")))]
    want = [run(g, *x, **kw) for x, kw in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(4):
        got = []
        for s, (x, kw) in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(run(g, *x, **kw))
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(u, w) for u, w in zip(a, b))


@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_offsets_beyond_32_bits(checkpoint):
    """Keys and values of more than 2^31 elements, read and written at both ends."""
    n, D = 8_500_000, 256
    assert n * D > 1 << 31
    src = torch.tensor([0, 1, n - 1, n - 2, n - 1, 5, n // 2, n - 3])
    dst = torch.tensor([0, 0, 0, 1, 1, 1, 2, 2])
    g = make_graph(src, dst, n, 3)
    used = torch.unique(src)
    small = torch.searchsorted(used, src)
    x = inputs(len(used), 3, 1, 1, D, torch.bfloat16, seed=3)
    k, v = (torch.zeros(n, 1, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    k[used.cuda()], v[used.cuda()] = x[1], x[2]
    got = run(g, x[0], k, v, x[3], checkpoint=checkpoint)
    h = make_graph(small, dst, len(used), 3)
    want = run(h, *x, checkpoint=checkpoint)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for a, b in zip(got[2:], want[2:]):
        assert torch.equal(a[used.cuda()], b)
        a[used.cuda()] = 0
        assert not a.any()


def test_copied_and_saved_graphs(tmp_path):
    """A graph is copied, and saved and loaded, with the items it keeps; they point at the copy's own arrays."""
    import copy
    from tango_amd.graph_attention import _items, prepare_attention
    x = inputs(300, 300, 2, 2, 16, torch.float32)
    g = prepare_attention(make_graph(*powerlaw_graph(np.random.default_rng(3), 300, 4000), 300, 300))
    want = run(g, *x)
    torch.save(g, tmp_path / "graph.pt")
    for other in (copy.copy(g), copy.deepcopy(g), torch.load(tmp_path / "graph.pt", weights_only=False)):
        kept = other._attention_items_in[2]
        assert _items(other, "in") is kept and kept.struct.indices == other.adj_csc32[0].data_ptr()
        got = run(other, *x)
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_a_graph_preprocessed_again_gets_new_items():
    from tango_amd.graph import Graph
    from tango_amd.graph_attention import graph_attention
    from tango_amd.util import graph_preprocess
    q, k, v, _ = inputs(4, 4, 1, 1, 8, torch.float32)
    g = graph_preprocess(Graph(torch.tensor([0, 1], device="cuda"), torch.tensor([2, 3], device="cuda"), 4))
    assert torch.equal(graph_attention(g, q, k, v)[2], v[0])
    g._src, g._dst, g._csr, g._csc = torch.tensor([3, 3], device="cuda"), torch.tensor([0, 1], device="cuda"), None, None
    out = graph_attention(graph_preprocess(g), q, k, v)
    assert torch.equal(out[0], v[3]) and (out[2] == 0).all()


def test_largest_scale():
    """2^127 is taken, with queries that bring the logits back; what times log2(e) leaves fp32's range is refused."""
    from tango_amd.graph_attention import graph_attention
    q, k, v, dout = inputs(20, 20, 2, 2, 16, torch.float32)
    g = make_graph(torch.arange(20).repeat(3), torch.arange(60) * 7 % 20, 20, 20)
    # a power of two moved between the factors, which times log2(e) changes no bit
    assert torch.equal(graph_attention(g, q * 2.0 ** -100, k, v, scale=2.0 ** 99), graph_attention(g, q, k, v, scale=0.5))
    assert torch.isfinite(graph_attention(g, q * 2.0 ** -100, k * 2.0 ** -27, v, scale=2.0 ** 127)).all()
    for scale in (1e39, -1e39, 3e38, 1e300):
        with pytest.raises(ValueError):
            graph_attention(g, q, k, v, scale=scale)


@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_kept_tensors_are_released_by_the_backward_pass(checkpoint):
    from tango_amd.graph_attention import graph_attention, prepare_attention
    # prepared, so that the backward pass leaves no new items (16 bytes a row) on the graph
    g = prepare_attention(make_graph(torch.arange(4000), torch.arange(4000), 4000, 4000))
    leaf = torch.randn(4000, 8, 32, device="cuda", requires_grad=True)
    q, k, v = (leaf * c for c in (1.0, 2.0, 3.0))  # nothing but the attention needs them
    out = graph_attention(g, q, k, v, checkpoint=checkpoint)
    del q, k, v
    loss = out.sum()
    before = torch.cuda.memory_allocated()
    loss.backward()
    # the gradient is new; all that was kept (a byte an element at least) is gone
    assert torch.cuda.memory_allocated() - before <= leaf.numel() * (4 - 3 * (1 if checkpoint else 4)) + 16384
    with pytest.raises(RuntimeError, match="second time"):
        loss.backward()


def test_refusals():
    from tango_amd.graph import Graph
    from tango_amd.graph_attention import graph_attention
    src, dst = torch.tensor([0, 1, 2]).cuda(), torch.tensor([0, 0, 1]).cuda()
    g = make_graph(src, dst, 3, 2)
    q, k, v, _ = inputs(3, 2, 4, 2, 8, torch.float32)
    graph_attention(g, q, k, v)
    ok = torch.ones(3, dtype=torch.bool, device="cuda")
    bad_runtime = [dict(q=q.double()), dict(k=k.bfloat16()), dict(q=q[0]), dict(q=k), dict(k=q[:, :2]), dict(v=v[:, :1]), dict(k=k[..., :4]),
                   dict(edge_mask=ok.float()), dict(edge_mask=ok[:2]), dict(edge_mask=ok.cpu()), dict(graph=Graph(src, dst, 3, 2))]
    bad_value = [dict(q=q[:, :3]), dict(checkpoint="int4"), dict(scale=float("nan")), dict(scale=float("inf")),
                 dict(q=torch.zeros(2, 1, 257, device="cuda"), k=torch.zeros(3, 1, 257, device="cuda"), v=torch.zeros(3, 1, 257, device="cuda"))]
    for kind, cases in ((RuntimeError, bad_runtime), (ValueError, bad_value)):
        for kw in cases:
            call = dict(graph=g, q=q, k=k, v=v)
            call.update(kw)
            with pytest.raises(kind):
                graph_attention(**call)


def test_changed_inputs_are_noticed():
    """An input changed in place between the passes is an error, as for torch's own operators; a checkpoint holds
    its own copy."""
    from tango_amd.graph_attention import graph_attention
    g = make_graph(np.array([0, 1]), np.array([1, 0]), 2, 2)
    q, k, v, dout = inputs(2, 2, 1, 1, 8, torch.float32)
    q.requires_grad_()
    out = graph_attention(g, q, k, v)
    k.mul_(2)
    with pytest.raises(RuntimeError):
        out.backward(dout)
    out = graph_attention(g, q, k, v, checkpoint="int8")
    k.mul_(2)
    out.backward(dout)
    assert q.grad is not None
