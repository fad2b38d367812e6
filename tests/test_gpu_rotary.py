"""rotate_axes and qk_norm_rotate against their formulas in 64 bits.

Tolerance, from the arithmetic: the store rounds by eps / 2 relative to the value (half the
smallest subnormal below that); before it, in fp32 (half steps of 2^-24), a turned value is
off by at most c * 2^-24 * (|a| + |b|) with its pair's two inputs a, b:
  rotation   the angle's rounding pi * 2^-25 * 2 turned into both terms (3.2), sine and cosine (2),
             two products and a sum (2): c = 8
  the norm   adds to a and b the sum of squares (8 serial terms and 5 shuffles, halved by the root:
             7), the mean and eps (1), the reciprocal root (4), two products (2): c = 8 + 16
"""
import pytest
import torch

from lithe_b200.kernels import qk_norm_rotate, rotate_axes

pytestmark = pytest.mark.gpu
DEV = "cuda"


def exact_turn(x, pos, axes, theta, pairing):
    """The turned values and, for the tolerance, |a| + |b| of every value's pair (fp64)."""
    x, pos = x.double(), pos.double()
    if pos.dim() == 2:
        pos = pos[None]
    ang = torch.cat([pos[..., i:i + 1] * torch.pow(torch.tensor(theta, dtype=torch.float64, device=x.device),
                                                   -torch.arange(0, d, 2, dtype=torch.float64, device=x.device) / max(d, 1))
                     for i, d in enumerate(axes)], -1)[:, :, None]
    r = 2 * ang.shape[-1]
    if pairing == "interleaved":
        a, b = x[..., 0:r:2], x[..., 1:r:2]
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
    u, v, m = a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin(), a.abs() + b.abs()
    if pairing == "interleaved":
        y, m = torch.stack([u, v], -1).flatten(-2), torch.stack([m, m], -1).flatten(-2)
    else:
        y, m = torch.cat([u, v], -1), torch.cat([m, m], -1)
    return torch.cat([y, x[..., r:]], -1), torch.cat([m, x[..., r:].abs()], -1)


def exact_norm(x, w, eps):
    x = x.double()
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    return y if w is None else y * w.double()


def check(got, want, scale, c):
    info = torch.finfo(got.dtype)
    half = 0.0 if got.dtype == torch.float32 else info.eps / 2
    tol = half * want.abs() + c * 2.0 ** -24 * scale + info.smallest_normal * info.eps
    err = (got.double() - want).abs()
    worst = (err - tol).max().item() if got.numel() else 0.0
    assert worst <= 0, f"off by {err.max().item()} (tolerance exceeded by {worst})"


def make(shape, dtype, seed=0, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pairing", ["interleaved", "halves"])
@pytest.mark.parametrize("b,s,h,d,axes", [
    (1, 1, 1, 2, (2,)), (1, 1, 24, 128, (16, 56, 56)), (2, 5, 3, 64, (16, 24, 24)), (3, 37, 4, 80, (16, 24, 24)),
    (2, 333, 24, 128, (16, 56, 56)), (1, 7, 5, 34, (10, 6)), (2, 9, 2, 256, (64, 64, 64, 64)), (1, 4, 33, 72, (8, 0, 64)),
    (1, 6, 1, 8, (2,)), (2, 3, 7, 20, (2, 2, 2, 2, 2, 2, 2, 2)), (1, 5001, 2, 40, (12, 14, 14))])
def test_rotation(b, s, h, d, axes, pairing, dtype):
    x = make((b, s, h, d), dtype)
    pos = torch.randint(-50, 500, (s, len(axes)), device=DEV, dtype=torch.int32)
    before = x.clone()
    got = rotate_axes(x, pos, axes, pairing=pairing)
    assert torch.equal(x, before) and got.is_contiguous() and got.dtype == dtype
    check(got, *exact_turn(x, pos, axes, 1e4, pairing), 8)
    again = x.clone()
    assert rotate_axes(again, pos, axes, pairing=pairing, out=again) is again
    assert torch.equal(again, got)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32])
@pytest.mark.parametrize("far", [1, 10 ** 4, 2 ** 24 - 1, 2 ** 31 - 1])
def test_far_and_own_positions(kind, far):
    b, s, h, d, axes = 2, 50, 3, 64, (32, 32)
    g = torch.Generator(device=DEV).manual_seed(far % 1000)
    pos = (torch.rand(b, s, 2, generator=g, device=DEV, dtype=torch.float64) * 2 - 1) * far
    pos = pos.to(kind)
    x = make((b, s, h, d), torch.float32, 3)
    for theta in (256.0, 1e6):
        check(rotate_axes(x, pos, axes, theta=theta), *exact_turn(x, pos, axes, theta, "interleaved"), 8)
    shared = rotate_axes(x, pos[1].contiguous(), axes)
    assert torch.equal(shared[1], rotate_axes(x, pos, axes)[1])


@pytest.mark.parametrize("pairing", ["interleaved", "halves"])
def test_strides_and_alignment(pairing):
    axes = (16, 24, 24)
    pos = torch.rand(11, 3, device=DEV) * 40
    fused = make((2, 11, 3, 5, 80), torch.bfloat16, 1)
    for part in range(3):
        x = fused[:, :, part]
        want = rotate_axes(x.contiguous(), pos, axes, pairing=pairing)
        assert torch.equal(rotate_axes(x, pos, axes, pairing=pairing), want)
        out = torch.zeros(2, 5, 11, 80, dtype=torch.bfloat16, device=DEV).transpose(1, 2)     # heads before tokens
        assert torch.equal(rotate_axes(x, pos, axes, pairing=pairing, out=out), want)
        flat = torch.zeros(want.numel() + 3, dtype=torch.bfloat16, device=DEV)
        for off in (1, 2, 3):                                            # bases off the 16-byte boundary
            odd = flat[off:off + want.numel()].view(want.shape)
            assert torch.equal(rotate_axes(x, pos, axes, pairing=pairing, out=odd), want)
            odd.copy_(x)
            assert torch.equal(rotate_axes(odd, pos, axes, pairing=pairing), want)
    rest = fused.clone()
    rotate_axes(rest[:, :, 1], pos, axes, pairing=pairing, out=rest[:, :, 1])
    assert torch.equal(rest[:, :, 0], fused[:, :, 0]) and torch.equal(rest[:, :, 2], fused[:, :, 2])
    expanded = make((1, 1, 5, 80), torch.bfloat16, 2).expand(2, 11, 5, 80)                    # an input may be expanded
    assert torch.equal(rotate_axes(expanded, pos, axes), rotate_axes(expanded.contiguous(), pos, axes))
    with pytest.raises(ValueError, match="overlaps"):
        rotate_axes(fused[:, :10, 0], pos[:10], axes, out=fused[:, 1:, 0])


@pytest.mark.parametrize("pairing", ["interleaved", "halves"])
def test_values_behind_the_pairs_are_copied(pairing):
    x = make((1, 6, 2, 64), torch.float32)
    x[..., 40:] = torch.tensor([float("nan"), float("inf"), -float("inf")] * 8, device=DEV)
    pos = torch.full((6, 1), 3.0, device=DEV)
    got = rotate_axes(x, pos, (40,), pairing=pairing)
    assert torch.equal(got[..., 40:].view(torch.int32), x[..., 40:].contiguous().view(torch.int32))
    assert torch.isfinite(got[..., :40]).all()


def test_no_tokens_and_bad_positions():
    x = torch.empty(2, 0, 3, 64, device=DEV)
    assert rotate_axes(x, torch.empty(0, 1, device=DEV), (64,)).shape == x.shape
    x = torch.empty(0, 4, 3, 64, device=DEV)
    assert rotate_axes(x, torch.empty(4, 1, device=DEV), (64,)).shape == x.shape
    x = make((1, 2, 3, 64), torch.float32)
    pos = torch.tensor([[float("nan"), 1.0], [float("inf"), 1.0]], device=DEV)
    got = rotate_axes(x, pos, (32, 32))                    # a bad position spoils its own axis of its own token
    assert got[..., :32].isnan().all() and torch.isfinite(got[..., 32:]).all()


def test_bad_positions_leave_the_values_that_stay():
    q = make((1, 2, 3, 64), torch.bfloat16, 1)
    pos = torch.tensor([[float("nan"), 1.0], [float("inf"), 1.0]], device=DEV)
    for pairing in ("interleaved", "halves"):
        got, _ = qk_norm_rotate(q, q, None, None, pos, (16, 8), pairing=pairing)
        fine, _ = qk_norm_rotate(q, q, None, None, torch.ones_like(pos), (16, 8), pairing=pairing)
        bad = torch.zeros(64, dtype=torch.bool, device=DEV)
        bad[:16] = True
        if pairing == "halves":
            bad[8:16], bad[12:20] = False, True
        assert got[..., bad].isnan().all() and torch.equal(got[..., ~bad], fine[..., ~bad])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pairing", ["interleaved", "halves"])
@pytest.mark.parametrize("b,s,h,kv,d,axes", [
    (1, 1, 1, 1, 128, (16, 56, 56)), (1, 1, 24, 24, 128, (16, 56, 56)), (2, 17, 8, 2, 64, (16, 24, 24)),
    (3, 130, 32, 8, 80, (40, 40)), (2, 700, 24, 24, 128, (16, 56, 56)), (1, 5, 3, 7, 256, (100,)), (2, 33, 5, 1, 72, (24, 24, 24)),
    (1, 3, 2, 2, 30, (4, 2)), (1, 2, 1, 1, 2, (2,))])
def test_norm_and_rotation(b, s, h, kv, d, axes, pairing, dtype):
    q, k = make((b, s, h, d), dtype, 1, 3.0), make((b, s, kv, d), dtype, 2, 0.1)
    wq, wk = 1 + make((d,), dtype, 3, 0.2), 1 + make((d,), dtype, 4, 0.2)
    pos = torch.rand(b, s, len(axes), device=DEV) * 100
    got_q, got_k = qk_norm_rotate(q, k, wq, wk, pos, axes, pairing=pairing)
    for got, x, w in ((got_q, q, wq), (got_k, k, wk)):
        check(got, *exact_turn(exact_norm(x, w, 1e-6), pos, axes, 1e4, pairing), 24)
    bare = qk_norm_rotate(q, k, None, None, pos, axes, pairing=pairing, eps=1e-3)
    check(bare[1], *exact_turn(exact_norm(k, None, 1e-3), pos, axes, 1e4, pairing), 24)
    wide = qk_norm_rotate(q, k, wq.float(), wk.float(), pos, axes, pairing=pairing)
    assert torch.equal(wide[0], got_q) and torch.equal(wide[1], got_k)
    iq, ik = q.clone(), k.clone()
    qk_norm_rotate(iq, ik, wq, wk, pos, axes, pairing=pairing, out_q=iq, out_k=ik)
    assert torch.equal(iq, got_q) and torch.equal(ik, got_k)


def test_joint_buffer_leaves_the_other_tokens():
    b, s, h, d, axes = 2, 21, 4, 128, (16, 56, 56)
    q, k = make((b, s, h, d), torch.bfloat16, 1), make((b, s, h, d), torch.bfloat16, 2)
    w = 1 + make((d,), torch.bfloat16, 3, 0.2)
    pos = torch.arange(s * 3, device=DEV).view(s, 3)
    want = qk_norm_rotate(q, k, w, w, pos, axes)
    joint = make((b, 60, 2, h, d), torch.bfloat16, 9)                    # q and k of the joint sequence in one buffer
    before = joint.clone()
    qk_norm_rotate(q, k, w, w, pos, axes, out_q=joint[:, 30:51, 0], out_k=joint[:, 30:51, 1])
    assert torch.equal(joint[:, 30:51, 0], want[0]) and torch.equal(joint[:, 30:51, 1], want[1])
    assert torch.equal(joint[:, :30], before[:, :30]) and torch.equal(joint[:, 51:], before[:, 51:])


def test_a_written_tensor_says_so():
    """torch's version counter of an output that the caller gave moves, as for any in-place write (the
    layers' shared preparations tell inputs apart by it)."""
    x = make((1, 3, 2, 64), torch.bfloat16, 1)
    pos = torch.zeros(3, 1, device=DEV)
    for write in (lambda: rotate_axes(x, pos, (64,), out=x), lambda: qk_norm_rotate(x, x.clone(), None, None, pos, (64,), out_q=x)):
        before = x._version
        write()
        assert x._version > before


def test_heads_do_not_meet():
    """A head of zeros stays zero, a head with a NaN or an infinity spoils only itself."""
    q = make((1, 3, 6, 64), torch.bfloat16, 1)
    clean = q.clone()
    q[0, 1, 2, 5], q[0, 1, 3] = float("nan"), 0.0
    pos = torch.rand(3, 2, device=DEV)
    got, _ = qk_norm_rotate(q, clean, None, None, pos, (32, 32))
    want, _ = qk_norm_rotate(clean, clean, None, None, pos, (32, 32))
    assert got[0, 1, 2].isnan().all() and (got[0, 1, 3] == 0).all()
    got[0, 1, 2:4] = want[0, 1, 2:4] = 0
    assert torch.equal(got, want)


def test_streams_and_graphs():
    b, s, h, d, axes = 2, 64, 8, 128, (16, 56, 56)
    q, k = make((b, s, h, d), torch.bfloat16, 1), make((b, s, 2, d), torch.bfloat16, 2)
    pos = torch.arange(s * 3, device=DEV, dtype=torch.int32).view(s, 3)
    want = qk_norm_rotate(q, k, None, None, pos, axes)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = qk_norm_rotate(q, k, None, None, pos, axes)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = qk_norm_rotate(q, k, None, None, pos, axes)
        turned = rotate_axes(held[0], pos, axes)
    new = make((b, s, h, d), torch.bfloat16, 7)
    q.copy_(new)
    pos.add_(5)
    graph.replay()
    torch.cuda.synchronize()
    again = qk_norm_rotate(new, k, None, None, pos, axes)
    assert torch.equal(held[0], again[0]) and torch.equal(held[1], again[1])
    assert torch.equal(turned, rotate_axes(again[0], pos, axes))


def test_views_beyond_32_bits():
    """A token behind the first 2^31 elements of its buffer."""
    h, d = 2, 64
    tokens = 2 ** 31 // (h * d) + 3
    buf = torch.empty(1, tokens, h, d, dtype=torch.bfloat16, device=DEV)
    x = buf[:, -4:]
    x.copy_(make((1, 4, h, d), torch.bfloat16, 4))
    pos = torch.rand(4, 2, device=DEV) * 9
    want = rotate_axes(x.clone(), pos, (32, 32))
    assert torch.equal(rotate_axes(x, pos, (32, 32), out=x), want)


def test_compiled_calls():
    pos = torch.arange(30, device=DEV).view(10, 3)
    q, k = make((1, 10, 4, 64), torch.bfloat16, 1), make((1, 10, 4, 64), torch.bfloat16, 2)

    def both(q, k):
        q, k = qk_norm_rotate(q, k, None, None, pos, (16, 24, 24))
        return rotate_axes(q, pos, (16, 24, 24)), k

    want = both(q, k)
    got = torch.compile(both, fullgraph=True, backend="aot_eager")(q, k)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_theta_and_axes_are_read_in_every_call():
    x, pos = make((1, 9, 2, 64), torch.float32, 1), torch.arange(18, device=DEV).view(9, 2)
    theta, axis = torch.tensor(1e4), torch.tensor(16)
    for t, a in ((1e4, 16), (256.0, 16), (256.0, 40)):
        theta.fill_(t)
        axis.fill_(a)
        assert torch.equal(rotate_axes(x, pos, (axis, 24), theta=theta), rotate_axes(x, pos, (a, 24), theta=t))
        q, _ = qk_norm_rotate(x, x, None, None, pos, (axis, 24), theta=theta)
        assert torch.equal(q, qk_norm_rotate(x, x, None, None, pos, (a, 24), theta=t)[0])


@pytest.mark.parametrize("kind", [torch.int64, torch.float32])
@pytest.mark.parametrize("far", [3, 1000, 10 ** 5])
def test_sines_and_cosines_hold_their_last_places(kind, far):
    """The pair (1, 0) gives the angle's cosine and sine.  They are within 3 half steps of fp32 of the value,
    also where they are near zero: the sine and cosine of the fraction's fp32 part (2 half steps, a unit in the
    last place), the sum with its rest (1); the fp64 angles of both sides (frequency, product, reduction: 4 half
    steps of 2^-53 of the angle each); and 1e-14 for the rest's squares."""
    g = torch.Generator(device=DEV).manual_seed(far)
    dim, theta, s = 256, 1e4, 20000
    pos = (torch.rand(s, 1, generator=g, device=DEV, dtype=torch.float64) * far).to(kind)
    x = torch.tensor([1.0, 0.0], device=DEV).repeat(dim // 2).expand(1, s, 1, dim)
    got = rotate_axes(x, pos, (dim,), theta=theta)[0, :, 0].double().view(s, dim // 2, 2)
    freq = torch.tensor([theta ** (-2.0 * i / dim) for i in range(dim // 2)], dtype=torch.float64, device=DEV)
    angle = pos.double() * freq
    for part, want in ((0, angle.cos()), (1, angle.sin())):
        tol = 3 * 2.0 ** -24 * want.abs() + 8 * 2.0 ** -53 * angle.abs() + 1e-14
        assert ((got[..., part] - want).abs() <= tol).all()
