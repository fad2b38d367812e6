"""quantize_rows and int8_linear against their formulas in 64 bits.

quantize_rows is exact: whole numbers and scales are compared for equality.  The linear's
tolerance, from the arithmetic: the store rounds by eps / 2 relative to the value; before it, in
fp32 (half steps of 2^-24), the sum of products is converted and scaled (its own rounding, the
activation scale's, two products: 4), and the bias and the expand's 16 terms are added by
additions that may truncate (2 half steps each: 34), each relative to at most the sum of
magnitudes of what is added: c = 40.
"""
import pytest
import torch

from lithe_b200 import _lib, device_errors
from lithe_b200.kernels import _launch, int8_linear, quantize_rows, quantize_weight

pytestmark = pytest.mark.gpu
DEV = "cuda"
NAN, INF = float("nan"), float("inf")


def make(shape, dtype, seed=0, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


def exact_rows(x):
    x = x.double()
    most = x.abs().amax(1, keepdim=True)
    q = torch.where(most > 0, torch.round(x * 127 / most), torch.zeros_like(x))
    return q, (most / 127).squeeze(1)


def exact_linear(x, w, ws, bias=None, h=None, b_dec=None):
    """(value, magnitude of what is added) in fp64."""
    q, s = exact_rows(x.flatten(0, -2))
    y = (q @ w.double().t()) * s[:, None] * ws.double()
    mag = y.abs()
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    if h is not None:
        hs = h.double().view(b_dec.shape[0], -1, 16)
        y = y + torch.bmm(hs, b_dec.double().transpose(1, 2)).reshape(y.shape)
        mag = mag + torch.bmm(hs.abs(), b_dec.double().abs().transpose(1, 2)).reshape(y.shape)
    return y.view(*x.shape[:-1], -1), mag.view(*x.shape[:-1], -1)


def check(got, want, mag):
    info = torch.finfo(got.dtype)
    tol = info.eps / 2 * want.abs() + 40 * 2.0 ** -24 * mag + info.smallest_normal * info.eps
    worst = ((got.double() - want).abs() - tol).max().item() if got.numel() else 0.0
    assert worst <= 0, worst
    assert device_errors() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_quotient_of_two_mantissas(dtype):
    """Rows whose maximum takes every mantissa, and in each row values of every mantissa down to
    half a step: all ties and all nearest misses of a tie there are."""
    bits = 8 if dtype == torch.bfloat16 else 11
    lead = torch.arange(2 ** (bits - 1), 2 ** bits, device=DEV, dtype=torch.float64)
    part = 128 if dtype == torch.bfloat16 else 64
    for first in range(0, lead.numel(), part):
        most = lead[first:first + part, None]
        cols = [most]
        for k in range(0, 10):
            v = (lead * 2.0 ** -k)[None].expand(most.shape[0], -1)
            cols.append(torch.where(v <= most, v, torch.zeros_like(v)) * (-1) ** k)
        x = (torch.cat(cols, 1) * 2.0 ** -bits).to(dtype)
        got = quantize_rows(x)
        q, s = exact_rows(x)
        assert torch.equal(got.q.double(), q) and torch.equal(got.scale, s.float())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 7), (2, 8), (5, 100), (4, 1000), (3, 1898), (7, 3072), (2, 8192), (3, 12288),
                                    (2, 15360), (2, 16392), (1, 131072)])
def test_rows(rows, k, dtype):
    x = make((rows, k), dtype, k, 3.0)
    got = quantize_rows(x)
    q, s = exact_rows(x)
    assert torch.equal(got.q.double(), q) and torch.equal(got.scale, s.float())
    assert got.q.stride(0) % 16 == 0 and got.shape == (rows,) and got.dtype == dtype
    wide = make((rows, k + 9), dtype, k)                                     # rows off the 16-byte boundaries
    assert torch.equal(quantize_rows(wide[:, 3:k + 3]).q, quantize_rows(wide[:, 3:k + 3].contiguous()).q)
    assert torch.equal(quantize_rows(x[:, None].expand(rows, 2, k)).q[::2], got.q)
    assert torch.equal(quantize_rows(x.t().contiguous().t()).q, got.q)       # a transposed layout


def test_extreme_rows():
    for dtype in (torch.bfloat16, torch.float16):
        info = torch.finfo(dtype)
        x = torch.zeros(8, 24, dtype=dtype, device=DEV)
        x[1, 3] = info.max
        x[1, 4] = -info.max
        x[2, 5], x[2, 6] = info.smallest_normal, -info.smallest_normal / 2
        x[3, 0], x[3, 1] = info.smallest_normal * info.eps, -info.smallest_normal * info.eps     # smallest subnormal
        x[4, 2], x[4, 3] = NAN, 1.0
        x[5, 2], x[5, 3] = INF, 1.0
        x[6, 2], x[6, 3] = -INF, NAN
        x[7] = -0.0
        got = quantize_rows(x)
        assert got.scale[4:7].isnan().all() and (got.q[4:7] == 0).all()
        fine = [0, 1, 2, 3, 7]
        q, s = exact_rows(x[fine])
        assert torch.equal(got.q[fine].double(), q) and torch.equal(got.scale[fine], s.float())


SHAPES = [(1, 1, 1), (1, 17, 64), (2, 40, 8), (4, 300, 4096), (4, 24, 4104), (3, 1091, 1000), (1, 16, 16384), (2, 3000, 136), (3, 16, 31), (7, 100, 130), (8, 264, 3072), (9, 256, 128), (14, 300, 1000), (16, 64, 16),
          (17, 512, 256), (31, 33, 65), (33, 1091, 200), (64, 256, 64), (100, 264, 1898), (127, 72, 400), (128, 256, 128),
          (129, 128, 4096), (200, 1091, 130), (255, 520, 512), (256, 256, 128), (257, 8, 1000), (300, 1000, 96),
          (513, 248, 640), (1000, 768, 1024), (1237, 1091, 1898), (2048, 3072, 320), (1, 3072, 12288), (14, 18432, 192)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,n,k", SHAPES)
def test_linear(rows, n, k, dtype):
    x = make((rows, k), dtype, rows + k)
    w, ws = quantize_weight(make((n, k), dtype, n, 0.02))
    bias = make((n,), dtype, 5) if rows % 2 else None
    got = int8_linear(x, w, ws, bias)
    assert got.shape == (rows, n) and got.dtype == dtype
    check(got, *exact_linear(x, w, ws, bias))
    assert torch.equal(int8_linear(quantize_rows(x), w, ws, bias), got)
    # rows do not meet: the first half alone gives the same bits
    half = (rows + 1) // 2
    check(int8_linear(x[:half], w, ws, bias), *exact_linear(x[:half], w, ws, bias))


@pytest.mark.parametrize("samples,rps,n,k", [(1, 1, 16, 64), (14, 1, 264, 128), (5, 3, 100, 130), (2, 16, 256, 64), (3, 24, 40, 96),
                                             (3, 100, 520, 256), (2, 128, 1091, 128), (7, 37, 256, 320), (4, 256, 512, 128),
                                             (14, 512, 768, 64), (2, 1000, 264, 100), (300, 1, 64, 64), (130, 5, 72, 64),
                                             (14, 256, 1536, 3072), (8, 1024, 1032, 320), (3, 2560, 1091, 1000),
                                             (2, 768, 3592, 520), (1, 7168, 712, 128), (5, 1280, 3000, 136),
                                             (5, 1000, 2000, 136), (20, 300, 1096, 1000)])
def test_expand(samples, rps, n, k):
    bf = torch.bfloat16
    x = make((samples, rps, k), bf, 1)
    w, ws = quantize_weight(make((n, k), bf, 2, 0.02))
    bias = make((n,), bf, 3)
    h, b_dec = make((samples * rps, 16), bf, 4), make((samples, n, 16), bf, 5, 0.1)
    got = int8_linear(x, w, ws, bias, h=h, b_dec=b_dec)
    assert got.shape == (samples, rps, n)
    check(got, *exact_linear(x, w, ws, bias, h, b_dec))
    # a sample whose factors are zero gets the base linear's bits, the others keep theirs
    b0 = b_dec.clone()
    b0[samples // 2] = 0
    other = int8_linear(x, w, ws, bias, h=h, b_dec=b0)
    base = int8_linear(x, w, ws, bias)
    assert torch.equal(other[samples // 2], base[samples // 2])
    keep = torch.arange(samples, device=DEV) != samples // 2
    assert torch.equal(other[keep], got[keep])


def test_bad_rows_stay_alone():
    """A row with an infinity or NaN is NaN throughout; a row of zeros is the bias; the others keep their bits."""
    for rows in (5, 40, 300):
        x = make((rows, 256), torch.bfloat16, 1)
        w, ws = quantize_weight(make((136, 256), torch.bfloat16, 2, 0.02))
        bias = make((136,), torch.bfloat16, 3)
        clean = int8_linear(x, w, ws, bias)
        y = x.clone()
        y[1, 7], y[2, 9], y[3] = NAN, -INF, 0
        got = int8_linear(y, w, ws, bias)
        assert got[1].isnan().all() and got[2].isnan().all() and torch.equal(got[3], bias)
        rest = [0] + list(range(4, rows))
        assert torch.equal(got[rest], clean[rest])


def test_largest_products():
    """All products of one sign at their largest: the int32 sums reach 127 * 127 * k."""
    for k in (4096, 131072):
        x = torch.ones(40, k, dtype=torch.bfloat16, device=DEV)
        w = torch.full((24, k), -127, dtype=torch.int8, device=DEV)
        got = int8_linear(x, w, torch.full((24,), 1.0 / 127, device=DEV))
        assert torch.equal(got.float(), torch.full((40, 24), -float(k), device=DEV).bfloat16().float())
    with pytest.raises(NotImplementedError):
        int8_linear(torch.ones(1, 131073, dtype=torch.bfloat16, device=DEV),
                    torch.zeros(1, 131088, dtype=torch.int8, device=DEV)[:, :131073], torch.ones(1, device=DEV))


def test_nothing_behind_the_rows_is_read_or_written():
    """k's remainder, rows and channels that end inside a tile: garbage behind them has no say, and
    the memory behind the result stays."""
    for rows, n, k in [(3, 20, 70), (40, 100, 200), (130, 264, 136), (300, 300, 200)]:
        x = make((rows, k), torch.bfloat16, 1)
        w, ws = quantize_weight(make((n, k), torch.bfloat16, 2, 0.02))
        want = int8_linear(x, w, ws)
        pad = -(-k // 16) * 16 + 32
        big = torch.full((n, pad), 113, dtype=torch.int8, device=DEV)
        big[:, :k] = w
        assert torch.equal(int8_linear(x, big[:, :k], ws), want)
        from lithe_b200.kernels import _launch
        rq = quantize_rows(x)
        qbig = torch.full((rows, pad), -77, dtype=torch.int8, device=DEV)
        qbig[:, :k] = rq.q
        space = torch.full((rows * n + 4096,), 7.0, dtype=torch.bfloat16, device=DEV)
        out = space[:rows * n].view(rows, n)
        _launch.int8_linear_(qbig[:, :k], rq.scale, big[:, :k], ws, None, out)
        assert torch.equal(out, want) and (space[rows * n:] == 7.0).all()
        odd = torch.full((rows * n + 1,), 7.0, dtype=torch.bfloat16, device=DEV)[1:].view(rows, n)
        _launch.int8_linear_(qbig[:, :k], rq.scale, big[:, :k], ws, None, odd)      # a base off the 16-byte boundary
        assert torch.equal(odd, want)


def test_no_rows_and_shapes():
    w, ws = quantize_weight(make((24, 64), torch.bfloat16, 2))
    assert int8_linear(torch.empty(0, 64, dtype=torch.bfloat16, device=DEV), w, ws).shape == (0, 24)
    assert int8_linear(torch.empty(2, 0, 64, dtype=torch.bfloat16, device=DEV), w, ws).shape == (2, 0, 24)
    x = make((2, 3, 64), torch.bfloat16, 4)
    assert torch.equal(int8_linear(x[0, 0], w, ws), int8_linear(x, w, ws)[0, 0])
    assert torch.equal(int8_linear(x.transpose(0, 1), w, ws), int8_linear(x, w, ws).transpose(0, 1))


def test_streams_and_graphs():
    for rows in (4, 40, 600):
        x = make((rows, 512), torch.bfloat16, 1)
        w, ws = quantize_weight(make((264, 512), torch.bfloat16, 2, 0.02))
        want = int8_linear(x, w, ws)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = int8_linear(x, w, ws)
        side.synchronize()
        assert torch.equal(got, want)
        graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            a = int8_linear(x, w, ws)
            a2 = int8_linear(x, w, ws)
        with torch.cuda.graph(other):
            b = int8_linear(x, w, ws)
        x.copy_(make((rows, 512), torch.bfloat16, 9))
        for _ in range(2):
            graph.replay()
            other.replay()
        torch.cuda.synchronize()
        want = int8_linear(x, w, ws)
        assert torch.equal(a, want) and torch.equal(a2, want) and torch.equal(b, want)


def test_two_streams_at_once():
    x = [make((700, 1024), torch.bfloat16, i) for i in range(2)]
    w, ws = quantize_weight(make((1032, 1024), torch.bfloat16, 2, 0.02))
    want = [int8_linear(v, w, ws) for v in x]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(int8_linear(x[i], w, ws))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


def test_compiled_call():
    w, ws = quantize_weight(make((40, 96), torch.bfloat16, 2))
    x = make((5, 96), torch.bfloat16, 1)
    fn = torch.compile(lambda t: int8_linear(t, w, ws), fullgraph=True, backend="aot_eager")
    assert torch.equal(fn(x), int8_linear(x, w, ws))


@pytest.mark.parametrize("k", [1, 7, 15, 127, 129, 384, 385, 392, 500, 1001, 2049, 4100, 8191, 8200, 16385, 20481])
def test_rows_from_any_element_on(k):
    """Rows from each of the 8 places in a 16-byte piece on, an odd stride apart, between NaNs that are not
    theirs; the bytes behind a row of q are left as they are."""
    rows = 5
    wide = torch.full((rows, (k + 20) | 1), NAN, dtype=torch.bfloat16, device=DEV)
    values = make((rows, k), torch.bfloat16, k)
    values[rows - 1, k - 1] = 9.0                   # the maximum as the last value
    want, scale = exact_rows(values)
    for at in range(9):
        wide.fill_(NAN)
        wide[:, at:at + k] = values
        q = torch.full((rows, (k + 15) // 16 * 16 + 16), 77, dtype=torch.int8, device=DEV)
        s = torch.empty(rows, device=DEV)
        _launch.quantize_rows_(wide[:, at:at + k], q[:, :k], s)
        assert torch.equal(q[:, :k].double(), want) and torch.equal(s, scale.float()), at
        assert bool((q[:, k:] == 77).all()), at
    many = values.repeat(500, 1)                    # 2500 rows: another split
    if k % 2:
        got = quantize_rows(many)
        assert torch.equal(got.q.double(), want.repeat(500, 1))


@pytest.mark.parametrize("samples,rps,n,k", [(8, 256, 1290, 200), (10, 100, 3000, 136), (1, 1000, 3001, 4096), (3, 768, 1160, 64)])
def test_one_pass_of_pairs(samples, rps, n, k):
    """Pair tiles that fill less than the GPU, chosen since the smaller tiles would take two passes."""
    for dtype in (torch.bfloat16, torch.float16):
        x = make((samples, rps, k), dtype, 1)
        w, ws = quantize_weight(make((n, k), dtype, 2, 0.02))
        bias = make((n,), dtype, 3)
        check(int8_linear(x, w, ws, bias), *exact_linear(x, w, ws, bias))
        space = torch.full((samples * rps * n + 512,), 7.0, dtype=dtype, device=DEV)
        out = space[:samples * rps * n].view(samples * rps, n)
        rows = quantize_rows(x)
        _launch.int8_linear_(rows.q, rows.scale, w, ws, bias, out)
        assert torch.equal(out.view(samples, rps, n), int8_linear(x, w, ws, bias))
        assert bool((space[samples * rps * n:] == 7.0).all())
        if dtype == torch.bfloat16:
            h, b_dec = make((samples * rps, 16), dtype, 4), make((samples, n, 16), dtype, 5, 0.1)
            check(int8_linear(x, w, ws, bias, h=h, b_dec=b_dec), *exact_linear(x, w, ws, bias, h, b_dec))


@pytest.mark.parametrize("samples,rps,n,k", [(7, 2, 40, 96), (7, 5, 72, 64), (7, 37, 256, 320), (3, 100, 520, 256), (5, 20, 264, 4096),
                                             (20, 300, 1096, 1000), (5, 1000, 2000, 136), (4, 256, 512, 128),
                                             (5, 1280, 3000, 136)])
def test_bad_factors_stay_with_their_sample(samples, rps, n, k):
    """A sample's decoded factors with infinities and NaN: its own rows have them in those channels, and every
    other value keeps its bits, on each of the kernel's paths (samples that end inside a tile among them)."""
    bf = torch.bfloat16
    x = make((samples, rps, k), bf, 1)
    w, ws = quantize_weight(make((n, k), bf, 2, 0.02))
    h, b_dec = make((samples * rps, 16), bf, 4), make((samples, n, 16), bf, 5, 0.1)
    clean = int8_linear(x, w, ws, h=h, b_dec=b_dec)
    for s in (0, samples // 2, samples - 1):
        b = b_dec.clone()
        b[s, 3, 7], b[s, 8], b[s, n - 1, 0] = INF, NAN, -INF
        got = int8_linear(x, w, ws, h=h, b_dec=b)
        bad = torch.zeros(samples, 1, n, dtype=torch.bool, device=DEV)
        bad[s, 0, [3, 8, n - 1]] = True
        bad = bad.expand_as(got)
        assert not got[bad].isfinite().any()
        assert torch.equal(got[~bad], clean[~bad]), s


@pytest.mark.parametrize("rows,n,k", [(2, 1091, 3072), (14, 264, 1000), (32, 256, 12288), (200, 520, 640), (3000, 1536, 512)])
def test_one_workspace_many_calls(rows, n, k):
    """Calls of other activations one behind the other through one workspace: each reads what its own
    quantisation has written, not what stood there."""
    xs = [make((rows, k), torch.bfloat16, i, 1.0 + i) for i in range(3)]
    w, ws = quantize_weight(make((n, k), torch.bfloat16, 9, 0.02))
    want = []
    for x in xs:
        q = quantize_rows(x)
        out = torch.empty(rows, n, dtype=torch.bfloat16, device=DEV)
        want.append(_launch.int8_linear_(q.q, q.scale, w, ws, None, out))
    space = torch.empty(_lib.lib().lithe_int8_workspace_bytes(rows, k), dtype=torch.uint8, device=DEV)
    got = [torch.empty_like(want[0]) for _ in range(30)]
    for i, out in enumerate(got):
        rc = _lib.lib().lithe_int8_linear_dynamic(
            xs[i % 3].data_ptr(), k, w.data_ptr(), w.stride(0), ws.data_ptr(), None, out.data_ptr(), _lib.DTYPE_BF16,
            rows, n, k, None, None, 0, 0, _launch.error_word(space.device).data_ptr(), space.data_ptr(),
            space.numel(), torch.cuda.current_stream().cuda_stream)
        assert rc == 0
    assert all(torch.equal(out, want[i % 3]) for i, out in enumerate(got))
    assert device_errors() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,k", [(64, 128), (1091, 1000), (3072, 320), (264, 4104), (1290, 12288)])
def test_a_row_has_the_same_bits_among_any_others(n, k, dtype):
    """The sums are exact and what follows is one expression everywhere, so a row does not depend on how many
    there are, that is on which kernel, tile or split takes it."""
    x = make((2300, k), dtype, 1)
    w, ws = quantize_weight(make((n, k), dtype, 2, 0.02))
    bias = make((n,), dtype, 3)
    whole = int8_linear(x, w, ws, bias)
    for rows in (1, 2, 8, 9, 16, 17, 40, 128, 129, 255, 600, 1100, 2048, 2299):
        assert torch.equal(int8_linear(x[:rows], w, ws, bias), whole[:rows]), rows
    assert torch.equal(int8_linear(x[1000:1003], w, ws, bias), whole[1000:1003])
