"""The attention over a graph's edges (with its gradient), the 8-bit checkpoints of activations, and what the backward
passes take from them, as measurable cases: inputs, one pass in a plain form or through this package's operators, and
the same outputs in 64 bits."""
import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    att = lambda name, **kw: dict(op="attention", name=name, **kw)
    return [
        # one mini-batch block (bipartite: few destinations, their sampled in-neighbours): the launch-bound end
        att("attention-block-fp32", src=2048, dst=512, edges=4096, loops=False, heads=4, kv_heads=4, dim=64, type="fp32",
            grad=True, mask=False, checkpoint=False),
        # a citation graph of PubMed's size under an HGT layer of 8 heads in bf16
        att("attention-pubmed-bf16", src=19717, dst=19717, edges=177302, loops=True, heads=8, kv_heads=8, dim=32,
            type="bf16", grad=True, mask=False, checkpoint=False),
        # ogbn-arxiv's size under the default HGT layer (hidden 256, 8 heads) in the package's own precision
        att("attention-arxiv-fp32", src=169343, dst=169343, edges=1166243, loops=True, heads=8, kv_heads=8, dim=32,
            type="fp32", grad=True, mask=False, checkpoint=False),
        # the three heads of 250 columns of the arxiv attention stack, rows that no 16-byte load divides
        att("attention-arxiv-wide-fp16", src=169343, dst=169343, edges=1166243, loops=True, heads=3, kv_heads=3, dim=250,
            type="fp16", grad=True, mask=False, checkpoint=False),
        # the share of Reddit's edges that link prediction trains on: many edges a row, hubs of thousands
        att("attention-reddit8-bf16", src=232965, dst=232965, edges=9168000, loops=True, heads=8, kv_heads=8, dim=32,
            type="bf16", grad=True, mask=False, checkpoint=False),
        # evaluation (no gradient) with dropped edges and keys shared by four heads each
        att("attention-amazon-eval-fp32", src=410236, dst=410236, edges=4878874, loops=True, heads=8, kv_heads=2, dim=32,
            type="fp32", grad=False, mask=True, checkpoint=False),
        # training that keeps queries, keys and values in 8 bits between the passes
        att("attention-checkpoint-pubmed-fp32", src=19717, dst=19717, edges=177302, loops=True, heads=8, kv_heads=8, dim=32,
            type="fp32", grad=True, mask=False, checkpoint=True),
        att("attention-checkpoint-arxiv-fp32", src=169343, dst=169343, edges=1166243, loops=True, heads=4, kv_heads=4,
            dim=64, type="fp32", grad=True, mask=False, checkpoint=True),
        # an activation put into 8 bits by the forward pass and read back by the backward pass: hidden features with
        # a scale for each head's columns, input features with one scale a row
        dict(op="pack", name="pack-arxiv-hidden-fp32", rows=169343, cols=256, group=32, type="fp32"),
        dict(op="pack", name="pack-reddit-input-bf16", rows=232965, cols=602, group=0, type="bf16"),
        # the gradients of a linear layer's weight and bias from its input's checkpoint
        dict(op="weight_grad", name="weight-grad-reddit-fp32", rows=232965, out=256, cols=602, group=0, type="fp32"),
        dict(op="weight_grad", name="weight-grad-pubmed-bf16", rows=19717, out=256, cols=500, group=128, type="bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "checkpoint", "pack", "weight_grad"])
    dtype = rng.choice(sorted(_TYPES))
    if kind in ("attention", "checkpoint"):
        dst = _log(rng, 1, 200000)
        square = rng.random() < 0.6
        src = dst if square else _log(rng, 1, 200000)
        kv = rng.randint(1, 4)
        heads = kv * rng.choice([1, 1, 2, 4])
        dim = rng.choice([8, 16, 32, 64, 128, rng.randint(1, 256)])
        # no more than the work of the largest listed case: 9.4 M edges of 256 columns
        edges = _log(rng, 1, max(2, min(4000000, 1000000000 // (heads * dim))))
        return dict(op="attention", src=src, dst=dst, edges=edges, loops=square, heads=heads, kv_heads=kv, dim=dim,
                    type=dtype, grad=kind == "checkpoint" or rng.random() < 0.7, mask=rng.random() < 0.4,
                    checkpoint=kind == "checkpoint")
    if kind == "pack":
        return dict(op="pack", rows=_log(rng, 1, 230000), cols=rng.choice([128, 256, rng.randint(1, 640)]),
                    group=rng.choice([0, 16, 32, 64, 128, rng.randint(1, 300)]), type=dtype)
    return dict(op="weight_grad", rows=_log(rng, 1, 230000), out=rng.choice([16, 64, 256, rng.randint(1, 300)]),
                cols=rng.choice([128, 256, 500, rng.randint(1, 640)]), group=rng.choice([0, 64, 128, 256]), type=dtype)


def _edges(case, gen):
    """Seeded edges with a power law at both ends: the endpoint at rank r of n is drawn with a density that falls as
    r^-0.6, ranks are dealt to the nodes at random."""
    def ends(n):
        rank = (torch.rand(case["edges"], generator=gen, device="cuda", dtype=torch.float64).pow(2.5) * n).long().clamp_(max=n - 1)
        return torch.randperm(n, generator=gen, device="cuda")[rank]

    src, dst = ends(case["src"]), ends(case["dst"])
    if case["loops"]:
        own_id = torch.arange(case["src"], device="cuda")
        src, dst = torch.cat([src, own_id]), torch.cat([dst, own_id])
    return src, dst


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = _TYPES[case["type"]]
    rand = lambda *shape: torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)
    state = {"case": case}
    if case["op"] == "attention":
        H, KV, D = case["heads"], case["kv_heads"], case["dim"]
        src, dst = _edges(case, gen)
        state.update(src=src, dst=dst, scale=1.0 / math.sqrt(D),
                     q=(1.5 * rand(case["dst"], H, D)).to(dtype), k=rand(case["src"], KV, D).to(dtype),
                     v=rand(case["src"], KV, D).to(dtype), dout=rand(case["dst"], H, D).to(dtype),
                     mask=torch.rand(src.numel(), generator=gen, device="cuda") < 0.7 if case["mask"] else None)
        if own:
            from tango_amd.graph import Graph
            from tango_amd.util import graph_preprocess
            bipartite = None if case["loops"] else case["dst"]
            state["graph"] = graph_preprocess(Graph(src, dst, case["src"], bipartite))
            if case["grad"]:
                for name in "qkv":
                    state[name].requires_grad_()
        return state
    # activations: rows of different magnitude, a few far values
    x = rand(case["rows"], case["cols"]) * torch.exp(rand(case["rows"], 1))
    x = torch.where(rand(case["rows"], case["cols"]) > 3.0, 8.0 * x, x).to(dtype)
    if case["op"] == "pack":
        state["x"] = x
        return state
    state["dy"] = (rand(case["rows"], case["out"]) * 0.01).to(dtype)
    if own:
        from tango_amd.checkpoint import pack
        state["packed"] = pack(x, group=case["group"] or None)
    else:
        state["q"], state["scales"] = _quantize(x, case["group"] or x.size(1))
        state["group"] = case["group"] or x.size(1)
    return state


def _quantize(x, group):
    """(whole numbers in -127 .. 127, scales): per run of ``group`` columns of a row (the last run may be shorter) the
    integer nearest to 127 x / max|x|, ties to even, and max|x| / 127 in fp32.  A run that holds an infinity or NaN has
    the scale NaN and zeros; a run of zeros has the scale 0."""
    rows, cols = x.shape
    n = (cols + group - 1) // group
    wide = torch.zeros(rows, n * group, dtype=torch.float64, device=x.device)  # ties are exact in 64 bits
    wide[:, :cols] = x
    wide = wide.view(rows, n, group)
    top = wide.abs().amax(2)
    ok = torch.isfinite(top) & (top > 0)
    q = torch.where(ok[:, :, None], torch.round(wide * 127.0 / torch.where(ok, top, 1.0)[:, :, None]), 0.0)
    scale = torch.where(torch.isfinite(top), top.float() / 127.0, float("nan"))
    return q.view(rows, n * group)[:, :cols].to(torch.int8), scale


def _restore(q, scale, group):
    return q.float() * scale.repeat_interleave(group, 1)[:, :q.size(1)]


def _restored(x):
    n, heads, dim = x.shape
    return _restore(*_quantize(x.reshape(n, heads * dim), dim), dim).view(n, heads, dim)


def _attention(s, q, k, v, dout=None):
    """softmax over the in-edges of each destination of scale * (q . k), times v; with ``dout`` also the gradients."""
    src, dst = s["src"], s["dst"]
    if s["mask"] is not None:
        src, dst = src[s["mask"]], dst[s["mask"]]
    n, H, D = q.shape
    rep = H // k.size(1)
    qe, ke, ve = q[dst], k[src].repeat_interleave(rep, 1), v[src].repeat_interleave(rep, 1)
    logit = (qe * ke).sum(2) * s["scale"]
    top = torch.full((n, H), -math.inf, device=q.device).scatter_reduce(0, dst[:, None].expand(-1, H), logit, "amax")
    p = torch.exp(logit - top[dst])
    total = torch.zeros((n, H), device=q.device).index_add_(0, dst, p)
    p = p / total[dst]
    if dout is None:
        return torch.zeros_like(q).index_add_(0, dst, ve.mul_(p[:, :, None]))
    de = dout[dst]
    dp = (de * ve).sum(2)
    delta = torch.zeros((n, H), device=q.device).index_add_(0, dst, p * dp)
    ds = (p * (dp - delta[dst]) * s["scale"])[:, :, None]
    dq = torch.zeros_like(q).index_add_(0, dst, ke.mul_(ds))
    shared = lambda e: torch.zeros_like(k).index_add_(0, src, e.view(-1, H // rep, rep, D).sum(2))
    return dq, shared(qe.mul_(ds)), shared(de.mul_(p[:, :, None]))


def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    dtype = _TYPES[case["type"]]
    if case["op"] == "attention":
        q, k, v = (state[name].float() for name in "qkv")
        out = _attention(state, q, k, v).to(dtype)
        if not case["grad"]:
            return [out]
        if case["checkpoint"]:
            q, k, v = _restored(q), _restored(k), _restored(v)
        return [out] + [g.to(dtype) for g in _attention(state, q, k, v, state["dout"].float())]
    if case["op"] == "pack":
        group = case["group"] or case["cols"]
        return [_restore(*_quantize(state["x"], group), group).to(dtype)]
    dy = state["dy"].float()
    x = _restore(state["q"], state["scales"], state["group"])
    return [torch.matmul(dy.t(), x).to(dtype), dy.sum(0).to(dtype)]


def _run_own(state, case):
    if case["op"] == "attention":
        from tango_amd.graph_attention import graph_attention
        qkv = state["q"], state["k"], state["v"]
        out = graph_attention(state["graph"], *qkv, scale=state["scale"], edge_mask=state["mask"],
                              checkpoint="int8" if case["checkpoint"] else None)
        if not case["grad"]:
            return [out]
        return [out.detach(), *torch.autograd.grad(out, qkv, state["dout"])]
    from tango_amd.checkpoint import pack, unpack, weight_grad
    if case["op"] == "pack":
        return [unpack(pack(state["x"], group=case["group"] or None))]
    return list(weight_grad(state["dy"], state["packed"], want_bias=True))


def work(case):
    size = 4 if case["type"] == "fp32" else 2
    if case["op"] == "attention":
        edges = case["edges"] + (case["src"] if case["loops"] else 0)
        wide, narrow = case["dst"] * case["heads"] * case["dim"], case["src"] * case["kv_heads"] * case["dim"]
        products = edges * case["heads"] * case["dim"] * 2
        arrays = 2 * wide + 2 * narrow  # q, out; k, v
        if case["grad"]:
            arrays *= 2  # dout, dq; dk, dv
        return {"bytes": size * arrays + 4 * edges + 8 * (case["dst"] + 1) + (edges if case["mask"] else 0),
                "flops": products * (7 if case["grad"] else 2)}
    groups = case["rows"] * -(-case["cols"] // (case["group"] or case["cols"]))
    held = case["rows"] * case["cols"] + 4 * groups  # the 8-bit values and their scales
    if case["op"] == "pack":
        return {"bytes": 2 * size * case["rows"] * case["cols"] + 2 * held, "flops": 3 * case["rows"] * case["cols"]}
    return {"bytes": size * (case["rows"] * case["out"] + case["out"] * (case["cols"] + 1)) + held,
            "flops": 2 * case["rows"] * case["out"] * case["cols"]}


def _exact_values(x, group):
    """The values that x's checkpoint stands for, run of columns by run of columns."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for c in range(0, x.size(1), group):
        part = x[:, c:c + group].double()
        top = part.abs().max(1, keepdim=True).values
        scale = (top / 127.0).float().double()  # held in fp32
        out[:, c:c + group] = torch.round(127.0 * part / torch.where(top > 0, top, 1.0)) * scale
    return out


def _exact_attention(s, h, rep, q, k, v):
    """One query head in 64 bits, as a function that autograd differentiates."""
    src, dst = s["src"], s["dst"]
    if s["mask"] is not None:
        kept = s["mask"].nonzero().squeeze(1)
        src, dst = src.index_select(0, kept), dst.index_select(0, kept)
    score = torch.einsum("ed,ed->e", q[:, h].index_select(0, dst), k[:, h // rep].index_select(0, src)) * s["scale"]
    weight = score.exp()  # scores stay within a few hundred: no shift needed in 64 bits
    weighted = v[:, h // rep].index_select(0, src) * weight[:, None]
    total = torch.zeros(q.size(0), dtype=torch.float64, device=q.device).index_add(0, dst, weight)
    summed = torch.zeros(q.size(0), q.size(2), dtype=torch.float64, device=q.device).index_add(0, dst, weighted)
    return summed / torch.where(total > 0, total, 1.0)[:, None]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "pack":
        return [_exact_values(s["x"], case["group"] or case["cols"])]
    if case["op"] == "weight_grad":
        dy = s["dy"].double()
        if own:
            held, scales, group = s["packed"].values, s["packed"].scale, s["packed"].group
        else:
            held, scales, group = s["q"], s["scales"], s["group"]
        column = torch.arange(case["cols"], device=dy.device) // group
        x = held.double() * scales.double()[:, column]
        return [dy.t() @ x, dy.sum(0)]
    H, rep = case["heads"], case["heads"] // case["kv_heads"]
    exactly = [s[name].detach().double() for name in "qkv"]
    out = torch.stack([_exact_attention(s, h, rep, *exactly) for h in range(H)], 1)
    if not case["grad"]:
        return [out]
    if case["checkpoint"]:
        exactly = [_exact_values(x.reshape(x.size(0), -1), case["dim"]).view_as(x) for x in exactly]
    leaves = [x.requires_grad_() for x in exactly]
    grads = [torch.zeros_like(x) for x in leaves]
    for h in range(H):  # one head at a time: a head's edge tensors are freed before the next one's
        o = _exact_attention(s, h, rep, *leaves)
        for total, part in zip(grads, torch.autograd.grad(o, leaves, s["dout"][:, h].double())):
            total += part
    return [out.detach()] + grads
