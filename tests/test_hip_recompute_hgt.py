"""The HGT layer on the recomputing attention, with and without 8-bit checkpoints: the operators together, as a model
uses them."""
import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def graph():
    from tango_amd.graph import chung_lu
    from tango_amd.util import graph_preprocess
    return graph_preprocess(chung_lu(1500, 20000, 2.1, seed=3, symmetric=True, device="cuda"))


def layer_pair(in_dim, out_dim, heads, **kw):
    from tango_amd.gat import HGTLayer
    torch.manual_seed(0)
    a = HGTLayer(in_dim, out_dim, heads).cuda()
    b = HGTLayer(in_dim, out_dim, heads, **kw).cuda()
    b.load_state_dict(a.state_dict())
    return a, b


def step(layer, graph, x, dy):
    x = x.clone().requires_grad_()
    y = layer(graph, x)
    return [y.detach(), *torch.autograd.grad(y, [x, *layer.parameters()], dy)]


@pytest.mark.parametrize("checkpoint", [None, "int8"])
def test_close_to_the_quantized_chain(graph, checkpoint):
    """Same parameters: the int8 chain rounds every operand to 1/254 of its tensor's range at most, the recomputing
    layer does not; both are the same function up to that (the outputs' scale is about 1, errors of a few percent)."""
    a, b = layer_pair(64, 128, 4, attention="recompute", checkpoint=checkpoint)
    gen = torch.Generator().manual_seed(1)
    x, dy = torch.randn(1500, 64, generator=gen).cuda(), torch.randn(1500, 128, generator=gen).cuda()
    names = ["out", "x"] + [n for n, _ in a.named_parameters()]
    for name, u, w in zip(names, step(a, graph, x, dy), step(b, graph, x, dy)):
        assert u.shape == w.shape and torch.isfinite(w).all()
        if name in ("k_linear.bias", "attn_linear.bias"):
            # a vector added to every key adds q . b to all logits of a row, which its softmax does not see: these
            # gradients are zero but for rounding, in both
            continue
        # a whole tensor's deviation against its own size: about 1 or more if a term were missing or of the wrong sign
        assert (u - w).norm() <= 0.25 * u.norm(), name


def test_gradients_are_the_formulas(graph):
    """What the layer hands its projections is the gradient of the softmax attention at its own projections."""
    from tango_amd.graph_attention import graph_attention
    from test_hip_graph_attention import check, formulas
    gen = torch.Generator().manual_seed(2)
    q, k, v, dout = (torch.randn(1500, 4, 32, generator=gen).cuda() for _ in range(4))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = graph_attention(graph, *leaves, scale=0.2)
    src, dst = graph.edges()
    check([out, *torch.autograd.grad(out, leaves, dout)], *formulas(src, dst, q, k, v, dout, 0.2, None), torch.float32)


def test_stack_with_a_checkpointed_read_out(graph):
    """Layers, checkpoints and a checkpointed linear read-out in one training step; twice the same bits."""
    from tango_amd.checkpoint import CheckpointLinear
    from tango_amd.gat import HGTStack
    from tango_amd.loss import cross_entropy

    def run():
        torch.manual_seed(5)
        model = HGTStack(64, 64, 7, 4, 2, attention="recompute", checkpoint="int8").cuda()
        model.proj = CheckpointLinear(64, 7, group=32).cuda()
        gen = torch.Generator().manual_seed(6)
        x, labels = torch.randn(1500, 64, generator=gen).cuda(), torch.randint(0, 7, (1500,), generator=gen).cuda()
        loss = cross_entropy(model(graph, x), labels)
        loss.backward()
        grads = [p.grad for p in model.parameters()]
        assert all(g is not None and torch.isfinite(g).all() and (g != 0).any() for g in grads)
        return [loss.detach(), *grads]

    assert all(torch.equal(a, b) for a, b in zip(run(), run()))


def test_kept_memory(graph):
    """Between the passes the checkpointed layer holds less than the plain one, which holds less than the chain."""
    from tango_amd.gat import HGTLayer
    held = {}
    x = torch.randn(1500, 256, device="cuda")
    for name, kw in (("chain", {}), ("recompute", dict(attention="recompute")), ("int8", dict(attention="recompute", checkpoint="int8"))):
        torch.manual_seed(0)
        layer = HGTLayer(256, 256, 8, **kw).cuda()
        layer(graph, x)  # plans, workspaces
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = layer(graph, x)
        held[name] = torch.cuda.memory_allocated() - before
        del y
    assert held["int8"] < held["recompute"]


def test_kept_tensors_on_the_host(graph):
    """torch's hooks on saved tensors see what is kept: offloaded to the host and back, the gradients are the same."""
    from tango_amd.checkpoint import CheckpointLinear
    from tango_amd.gat import HGTLayer
    torch.manual_seed(9)
    layer = HGTLayer(64, 64, 2, attention="recompute", checkpoint="int8").cuda()
    proj = CheckpointLinear(64, 7, group=32).cuda()
    x, dy = torch.randn(1500, 64, device="cuda"), torch.randn(1500, 7, device="cuda")
    leaves = [*layer.parameters(), *proj.parameters()]
    want = torch.autograd.grad(proj(layer(graph, x)), leaves, dy)
    with torch.autograd.graph.save_on_cpu():
        y = proj(layer(graph, x))
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(y, leaves, dy)))


def test_training_driver(capsys):
    from tango_amd.evaluation import train
    for checkpoint in (None, "int8"):
        ms, loss = train("hgt", "pubmed", epochs=4, quiet=True, attention="recompute", checkpoint=checkpoint)
        assert ms > 0 and loss == loss
    with pytest.raises(ValueError):
        train("gcn", "pubmed", epochs=1, quiet=True, attention="recompute")


def test_refusals():
    from tango_amd.gat import HGTLayer
    for kw in (dict(attention="fused"), dict(checkpoint="int8"), dict(attention="recompute", checkpoint="fp8")):
        with pytest.raises(ValueError):
            HGTLayer(8, 8, 2, **kw)
