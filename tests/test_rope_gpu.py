"""rope.apply on the GPU against a float64 evaluation with the same tables. Tolerance of an element: each product and
the sum are rounded to fp32 (3 * 2^-24 of |x0 c| + |x1 s|), then once to the output type (half a step of the value)."""
import pytest
import torch

from tests import _paged as P

pytestmark = pytest.mark.gpu


def check(y, x, table, rows, inverse=False):
    ref, size = P.rotate(x.cpu().double(), table.cos.cpu(), table.sin.cpu(), rows.cpu(), table.interleaved, inverse)
    # below the normal range of the type a step is its smallest subnormal
    tiny = torch.finfo(y.dtype).smallest_normal * torch.finfo(y.dtype).eps
    tol = 3 * 2.0 ** -24 * size + torch.finfo(y.dtype).eps / 2 * ref.abs() * (1 + 2.0 ** -20) + tiny
    err = (y.cpu().double() - ref).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("interleaved", [True, False], ids=["pairs", "half"])
@pytest.mark.parametrize("b,l,h,hk,d,rot", [(1, 1, 1, 0, 128, 128), (3, 17, 5, 2, 128, 64), (2, 5, 24, 12, 128, 128),
                                            (1, 7, 3, 1, 40, 10), (2, 3, 1, 1, 2, 2), (1, 4, 2, 2, 512, 480)])
def test_matches_float64(b, l, h, hk, d, rot, interleaved, dtype):
    from lingbot_b200 import rope
    g = torch.Generator().manual_seed(b + 10 * l + rot)
    table = rope.tables(200000, rot, interleaved=interleaved)
    x = torch.randn(b, l, h, d, generator=g).to(dtype).cuda()
    rows = torch.randint(0, 200000, (b, l), generator=g).cuda()
    if hk == 0:
        check(rope.apply(x, table, rows), x, table, rows)
        return
    k = torch.randn(b, l, hk, d, generator=g).to(dtype).cuda()
    y, z = rope.apply(x, table, rows.int(), k=k)
    check(y, x, table, rows)
    check(z, k, table, rows)


@pytest.mark.parametrize("interleaved", [True, False], ids=["pairs", "half"])
def test_strides_in_place_and_start(interleaved):
    """Views of a fused projection, one odd channel offset, in place, positions from `start` and shared by the batch."""
    from lingbot_b200 import rope
    table = rope.tables(500, 64, interleaved=interleaved)
    base = torch.randn(2, 9, 6, 3 * 128 + 1, generator=torch.Generator().manual_seed(0)).bfloat16().cuda()
    rows = (torch.arange(9) + 77).expand(2, 9)
    for lo in (0, 128, 257):                                  # 257: not 16-byte aligned
        x = base[:, :, :, lo:lo + 128]
        check(rope.apply(x, table, start=77), x, table, rows)
    y = base.clone()
    x = y[:, :, :, 128:256]
    got = rope.apply(x, table, rows[0].cuda(), out=x)
    assert got.data_ptr() == x.data_ptr()
    check(y[:, :, :, 128:256], base[:, :, :, 128:256], table, rows)
    assert torch.equal(y[:, :, :, :128], base[:, :, :, :128]) and torch.equal(y[:, :, :, 256:], base[:, :, :, 256:])
    e = base[:1, :, :, :128].expand(2, 9, 6, 128)             # broadcast input
    check(rope.apply(e, table, start=77), e, table, rows)


def test_inverse_is_the_gradient():
    """<apply(x), g> has the gradient apply(g, inverse=True): against the float64 transpose, and against differences."""
    from lingbot_b200 import rope
    g = torch.Generator().manual_seed(3)
    table = rope.tables(1000, 96, base=500.0, interleaved=False)
    x, w = (torch.randn(2, 4, 3, 128, generator=g).cuda() for _ in range(2))
    rows = torch.randint(0, 1000, (2, 4), generator=g).cuda()
    grad = rope.apply(w, table, rows, inverse=True)
    check(grad, w, table, rows, inverse=True)
    for at in [(0, 0, 0, 0), (1, 3, 2, 50), (0, 2, 1, 127)]:
        e = torch.zeros_like(x)
        e[at] = 0.5
        hi = (rope.apply(x + e, table, rows).double() * w.double()).sum()
        lo = (rope.apply(x - e, table, rows).double() * w.double()).sum()
        # linear: the difference quotient is exact but for fp32 roundings of about 4 terms of size |x| |w| each way
        assert abs(float(hi - lo) - float(grad[at])) <= 16 * 2.0 ** -23 * float(x.abs().max() * w.abs().max() + 1)


@pytest.mark.parametrize("scaling,pos", [({"type": "linear", "factor": 8}, 100000), ({"type": "ntk", "factor": 4}, 60000),
                                         ({"type": "banded", "factor": 4, "original": 8192, "low": 1, "high": 4}, 32000)])
def test_scaled_tables(scaling, pos):
    import math
    from lingbot_b200 import rope
    t = rope.tables(pos + 1, 128, scaling=scaling)
    for i in (0, 13, 40, 63):
        base = 10000.0 * (scaling["factor"] ** (128 / 126) if scaling["type"] == "ntk" else 1.0)
        f = base ** (-2 * i / 128)
        if scaling["type"] == "linear":
            f /= 8
        if scaling["type"] == "banded":
            keep = min(1.0, max(0.0, (8192 * f / (2 * math.pi) - 1) / 3))
            f = f / 4 * (1 - keep) + f * keep
        # fp32 rounding of the table, and 64-bit rounding of an angle up to 1e5
        assert abs(float(t.cos[pos, i]) - math.cos(pos * f)) <= 2.0 ** -24 + 1e-9
        assert abs(float(t.sin[pos, i]) - math.sin(pos * f)) <= 2.0 ** -24 + 1e-9


def test_position_outside_the_tables_is_recorded():
    from lingbot_b200 import _lib, rope
    table = rope.tables(16, 128)
    x = torch.randn(1, 3, 2, 128).bfloat16().cuda()
    y = rope.apply(x, table, torch.tensor([[3, 16, -1]], dtype=torch.int32).cuda())
    assert _lib.device_status() == 0x306
    check(y[:, :1], x[:, :1], table, torch.tensor([[3]]))
    assert torch.equal(y[:, 1:], x[:, 1:])


def test_other_stream_and_graph():
    from lingbot_b200 import rope
    table = rope.tables(64, 128)
    x = torch.randn(2, 8, 4, 128).half().cuda()
    rows = torch.arange(8, device="cuda").expand(2, 8)
    want = rope.apply(x, table, rows)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = rope.apply(x, table, rows)
    side.synchronize()
    assert torch.equal(got, want)
    y = torch.empty_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rope.apply(x, table, rows, out=y)
    x.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, rope.apply(x, table, rows))


def test_refusals():
    from lingbot_b200 import rope
    t = rope.tables(8, 64)
    x = torch.randn(1, 4, 2, 128, device="cuda")
    with pytest.raises(RuntimeError, match="gradient"):
        rope.apply(x.clone().requires_grad_(), t)
    with pytest.raises(Exception, match="rot"):
        rope.apply(x[..., :32].contiguous(), t)
    with pytest.raises(ValueError, match="shares memory"):
        rope.apply(x[:, :3], t, out=x[:, 1:])
    with pytest.raises(ValueError, match="positions"):
        rope.apply(x, t, torch.zeros(1, 3, dtype=torch.int32, device="cuda"))
    with pytest.raises(TypeError, match="positions"):
        rope.apply(x, t, torch.zeros(1, 4, device="cuda"))
    with pytest.raises(TypeError):
        rope.apply(x.double(), t)
    with pytest.raises(ValueError, match="does not go with"):
        rope.apply(x, t, k=x.half())
    with pytest.raises(ValueError, match="both or neither"):
        rope.apply(x, t, out=x, k=x.clone())
    with pytest.raises(ValueError, match="share memory"):
        rope.apply(x, t, out=torch.empty_like(x)[:, :1].expand(1, 4, 2, 128))
    with pytest.raises(ValueError, match="swapped"):
        y = x.clone()
        rope.apply(x, t, out=y, k=y, k_out=torch.empty_like(y))
    assert rope.apply(x[:, :0], t).shape == (1, 0, 2, 128)


def test_outputs_of_both_tensors_are_their_own_memory():
    """Q and K of one fused buffer rotate in place; one buffer for both results, or a result over the other's input, is
    refused."""
    from lingbot_b200 import rope
    table = rope.tables(64, 128)
    buf = torch.randn(2, 9, 5, 128, generator=torch.Generator().manual_seed(0)).bfloat16().cuda()
    q, k = buf[:, :, :3], buf[:, :, 3:]
    want = rope.apply(q, table, k=k)
    hold = torch.empty(2, 9, 5, 128, dtype=torch.bfloat16, device="cuda")
    one = torch.empty(2, 9, 3, 128, dtype=torch.bfloat16, device="cuda")
    flat = torch.empty(20000, dtype=torch.bfloat16, device="cuda")
    for x, y, out, k_out in ((q, k, one, one[:, :, :2]), (q, k, hold[:, :, :3], hold[:, :, 2:4]), (q, k, one, q[:, :, 1:]),
                             (q, k, k[:, :, :1].expand(q.shape), one[:, :, :2]), (buf[:, :, :4], buf[:, :, 3:], buf[:, :, :4], buf[:, :, 3:]),
                             (q, k, flat.as_strided(q.shape, (9 * 256, 256, 64, 1)), one[:, :, :2])):
        with pytest.raises(ValueError, match="share|swapped"):
            rope.apply(x, table, k=y, out=out, k_out=k_out)
    got = rope.apply(q, table, k=k, out=hold[:, :, :3], k_out=hold[:, :, 3:])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    got = rope.apply(q, table, k=k, out=q, k_out=k)
    assert torch.equal(got[0], want[0]) and torch.equal(buf[:, :, 3:], want[1])
