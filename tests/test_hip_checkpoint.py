"""8-bit checkpoints against their definition in exact arithmetic.

The integers are decided in 64 bits: 127 x is exact there (at most 31 bits), a quotient that is a tie is exact, and one
that is not differs from a tie by more than 2^-40 of itself, far more than a 64-bit division's rounding.  So integers
must be equal, scales are one fp32 division (equal), and a restored value is one product and one rounding (equal)."""
import math

import numpy as np
import pytest
import torch

from gpu_util import host

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
# the largest fp32 scale whose 127-fold does not overflow
LARGEST = np.float32(np.finfo(np.float32).max / 127.0)
LARGEST = LARGEST if float(LARGEST) * 127.0 <= float(np.finfo(np.float32).max) else np.nextafter(LARGEST, np.float32(0))


def expected(x, group):
    """(integers, scales) of a 2-D tensor, from the definition."""
    x = x.detach().cpu().double().numpy()
    rows, cols = x.shape
    q = np.zeros((rows, cols), np.int64)
    scale = np.zeros((rows, -(-cols // group)), np.float32)
    for j in range(scale.shape[1]):
        run = x[:, j * group:(j + 1) * group]
        with np.errstate(invalid="ignore", divide="ignore"):
            top = np.abs(run).max(1, initial=0.0)  # NaN if the run holds one
            good = np.isfinite(top)
            scale[:, j] = np.where(good, np.minimum(top.astype(np.float32) / np.float32(127), LARGEST), np.float32("nan"))
            live = good & (top > 0)
            n = np.rint(127.0 * run / np.where(live, top, 1.0)[:, None])  # half to even
        q[:, j * group:(j + 1) * group] = np.where(live[:, None], n, 0.0)
    return q, scale


def compare(x, group):
    from tango_amd.checkpoint import pack, unpack
    cols = x.size(-1)
    p = pack(x, group)
    q, scale = expected(x.reshape(math.prod(x.shape[:-1]), cols), group or max(cols, 1))
    assert p.values.dtype == torch.int8 and p.values.shape == q.shape
    assert np.array_equal(host(p.values), q)
    assert np.array_equal(host(p.scale), scale, equal_nan=True)
    spread = np.repeat(scale, group or max(cols, 1), axis=1)[:, :cols]
    with np.errstate(invalid="ignore"):
        value = torch.from_numpy(q.astype(np.float32) * spread).reshape(x.shape)
    for t in TYPES.values():
        y = unpack(p, t)
        assert y.dtype == t and y.shape == x.shape
        torch.testing.assert_close(y.cpu(), value.to(t), rtol=0, atol=0, equal_nan=True)
    assert unpack(p).dtype == x.dtype


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows,cols,group", [
    (1, 1, None), (1, 1, 1), (3, 5, 2), (7, 41, 41), (64, 256, 32), (65, 256, 256), (130, 602, None), (33, 500, 128),
    (19, 250, 250), (40, 96, 24), (5, 37, 8), (300, 16, 16), (9, 1000, 300), (4, 1025, None), (3, 5001, None), (2, 9000, 4500),
    (1000, 7, 1), (17, 64, 1000),
])
def test_against_the_definition(dtype, rows, cols, group):
    gen = torch.Generator().manual_seed(rows * 7919 + cols)
    x = torch.randn(rows, cols, generator=gen) * torch.exp(2 * torch.randn(rows, 1, generator=gen))
    compare(x.to(TYPES[dtype]).cuda(), group)


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_ties_go_to_even(dtype):
    """127 x / max|x| = n + 1/2 exactly for x = max|x| (2 n + 1) / 254; with max|x| = 254 * 2^e every such x is an odd
    multiple of 2^e, which all three types hold."""
    odd = torch.arange(-253, 254, 2, dtype=torch.float64)
    for e in (-14, -3, 0, 4):
        x = torch.cat([odd, torch.tensor([254.0], dtype=torch.float64)]) * 2.0 ** e
        compare(x.to(TYPES[dtype]).cuda()[None], None)
    half = torch.tensor([[1.3, 0.65, -0.65, 0.0, 1.3 / 4]]).to(TYPES[dtype])
    half[0, 1], half[0, 2] = half[0, 0] / 2, -half[0, 0] / 2  # 63.5 goes to 64
    compare(half.cuda(), None)


def test_next_to_ties_in_fp32():
    """Neighbours of ties: quotients one or a few fp32 steps off n + 1/2 on either side."""
    tops = torch.tensor([1.0, 1.5, 3.1415927, 0.7, 1e-30, 3e38, 1.1754944e-38, 2e-39, 254e-45], dtype=torch.float32)
    rows = []
    for top in tops:
        t = (top.double() * (2 * torch.arange(127, dtype=torch.float64) + 1) / 254).float()
        bits = t.view(torch.int32)
        near = torch.cat([(bits + k).clamp(min=0).view(torch.float32) for k in range(-3, 4)])
        near = torch.minimum(near, top)
        rows.append(torch.cat([near, top[None]]))
    x = torch.stack(rows)
    compare(x.cuda(), None)
    compare((-x).cuda(), None)


def test_extremes_and_missing_values():
    from tango_amd.checkpoint import pack, unpack
    inf, nan = float("inf"), float("nan")
    x = torch.zeros(9, 64)
    x[1, 3] = inf
    x[2, 5] = -inf
    x[3, 40] = nan
    x[4] = 3.4e38
    x[5, 0], x[5, 1] = torch.finfo(torch.float32).max, torch.finfo(torch.float32).min
    x[6] = torch.linspace(-1e-44, 1e-44, 64)  # subnormal scale
    x[7, 9] = 1e-45                           # its scale rounds to zero
    x[8, :32] = -0.0
    for group in (None, 32, 7, 1):
        compare(x.cuda(), group)
        assert torch.isfinite(unpack(pack(x[4:].cuda(), group))).all()
    for dtype in ("bf16", "fp16"):
        compare(x.clamp(-6e4, 6e4).to(TYPES[dtype]).cuda(), 16)


def test_layouts():
    """Views that are read in place or copied: row strides, columns off alignment, transposes, one broadcast row."""
    base = torch.randn(70, 300, generator=torch.Generator().manual_seed(5)).cuda()
    for x in (base[:, :256], base[:, 1:257], base[::2, 3:100], base.t(), base[:1].expand(70, 300), base[:, :1],
              base.view(10, 7, 300), base.view(10, 7, 300)[:, 1:3, :64], base[0], base[:0], base[:, :0]):
        compare(x, 32)
        compare(x.to(torch.bfloat16), None)


def test_many_runs():
    """More runs than a launch has lane groups, and the checkpoint's bytes."""
    from tango_amd.checkpoint import pack
    x = torch.randn(200_000, 48, generator=torch.Generator().manual_seed(2)).cuda()
    compare(x, 4)
    p = pack(x, 16)
    assert p.nbytes() == 200_000 * 48 + 4 * 200_000 * 3


def test_captured_and_replayed():
    """Both calls in one HIP graph, replayed over new inputs with eager work between the replays."""
    from tango_amd.checkpoint import pack, unpack
    x = torch.randn(500, 96, device="cuda")
    unpack(pack(x, 32))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = unpack(pack(x, 32))
    for _ in range(3):
        x.copy_(torch.randn(500, 96, device="cuda") * 3)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, unpack(pack(x, 32)))


def test_on_another_stream():
    from tango_amd.checkpoint import pack, unpack
    x = torch.randn(3000, 128, device="cuda")
    want = unpack(pack(x, 64))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = unpack(pack(x, 64))
    s.synchronize()
    assert torch.equal(got, want)


def test_saved_and_loaded(tmp_path):
    """A checkpoint travels: copied and loaded it unpacks to the same, on the host it is refused."""
    import copy
    from tango_amd.checkpoint import pack, unpack, weight_grad
    p = pack(torch.randn(40, 24, device="cuda"), 8)
    torch.save(p, tmp_path / "p.pt")
    load = lambda **kw: torch.load(tmp_path / "p.pt", weights_only=False, **kw)
    for q in (copy.copy(p), copy.deepcopy(p), load()):
        assert torch.equal(unpack(q), unpack(p))
    q = load(map_location="cpu")
    for call in (lambda: unpack(q), lambda: weight_grad(torch.ones(40, 3, device="cuda"), q)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_refusals():
    from tango_amd.checkpoint import pack, unpack
    x = torch.randn(4, 8, device="cuda")
    with pytest.raises(RuntimeError):
        pack(x.double())
    with pytest.raises(RuntimeError):
        pack(x[0, 0])
    for group in (0, -3, 2.5):
        with pytest.raises(ValueError):
            pack(x, group)
    with pytest.raises(RuntimeError):
        unpack(pack(x), torch.int8)
    with pytest.raises(TypeError):
        unpack(x)
