"""4-bit weights and 8-bit rows: packing, the norm and the activation that leave 8 bits, and the products, against their definitions
in 64 bits, at sizes off every tile and block and with values at the ends of their ranges."""
import pytest
import torch

import mx_util as U
from transformer_amd import kernels

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _gen(*key):
    return torch.Generator(device=DEV).manual_seed(sum(7919 ** i % 1000003 * int(v) for i, v in enumerate(key)))


def _randn(*shape, key=()):
    return torch.randn(*shape, generator=_gen(*shape, *key), device=DEV)


def _weights(n, k, seed=0):
    w = kernels.Mx4.empty(n, k, DEV)
    return kernels.mx4_pack(_randn(n, k, key=(seed, 4)) / k ** 0.5, w)


def _rows8(m, k, seed=0):
    x = _randn(m, k, key=(seed, 8)) * torch.exp(0.5 * _randn(k, key=(seed, 9)))
    return kernels.mx8_pack(x, kernels.Mx8.empty(m, k, DEV))


def _bits(t):
    return t.view(torch.uint8)


# ------------------------------------------------------------------ packing
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,k", [(1, 32), (3, 64), (33, 160), (257, 2080)])
def test_packing_gives_the_nearest_codes(n, k, dtype):
    wide = torch.full((n, k + 16), float("nan"), device=DEV, dtype=dtype)
    x = wide[:, 8:k + 8]
    x.copy_(_randn(n, k) * torch.exp2(torch.randint(-20, 20, (n, k // 32), generator=_gen(n, k), device=DEV).float()).repeat_interleave(32, 1))
    if n > 2:
        x[0, :32] = 0.0
        x[1, 32:64] = torch.arange(32, device=DEV).to(dtype) / 4 - 4          # every tie of the weights' grid, -4 to 3.75
        x[2, :32] = torch.tensor([1.0 + i / 16 for i in range(32)], device=DEV).to(dtype)
    y = x.double()
    rows = kernels.mx8_pack(x, kernels.Mx8.empty(n, k, DEV))
    want, b = U.pack8(y)
    assert torch.equal(rows.scales, b) and torch.equal(rows.codes.float().double(), want)
    w = kernels.mx4_pack(x, kernels.Mx4.empty(n, k, DEV))
    b = U.bytes_of(y, 6.0)
    s = U.power(b).repeat_interleave(32, 1)
    want = U.nearest(y / s, torch.tensor(U.E2M1, dtype=torch.float64, device=DEV)) * s
    assert torch.equal(w.scales, b) and torch.equal(U.values4(w.codes, w.scales), want)


def test_packing_at_the_ends_of_the_range():
    """Blocks at a border of two scales, of the smallest and largest numbers, of nothing, and with what is not finite."""
    tops = [448.0, 448.0001, 6.0, 6.000001, 1e-45, 2.0 ** -127, 2.0 ** -126, 2.0 ** -119, 3.4028234663852886e38, 1.0, 0.0, float("inf"), float("-inf"), float("nan")]
    x = torch.zeros(len(tops), 32, device=DEV)
    x[:, 5] = torch.tensor(tops, device=DEV)
    x[:, 6] = -x[:, 5] / 3
    x[-1, 6] = 1.0
    rows, w = kernels.mx8_pack(x, kernels.Mx8.empty(*x.shape, DEV)), kernels.mx4_pack(x, kernels.Mx4.empty(*x.shape, DEV))
    want, b = U.pack8(x.double())
    assert torch.equal(rows.scales, b) and torch.equal(rows.codes.float().double().nan_to_num(9.0), want.nan_to_num(9.0))
    assert torch.equal(w.scales, U.bytes_of(x.double(), 6.0))
    got = U.values4(w.codes, w.scales)
    assert bool(got[11:].isnan().all()) and bool((w.codes[11:] == 0).all()) and bool(got[:11].isfinite().all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_unpacking_every_code_and_scale(dtype):
    codes = torch.arange(256, dtype=torch.uint8, device=DEV).repeat(256, 1)         # every byte, 16 bytes a block, under every scale
    scales = torch.arange(256, dtype=torch.uint8, device=DEV).unsqueeze(1).repeat(1, 16)
    w = kernels.Mx4(codes, scales)
    room = torch.full((257, 520), 7.0, device=DEV, dtype=dtype)
    kernels.mx4_unpack(w, room[:256, :512])
    want = U.values4(codes, scales).to(dtype)
    assert torch.equal(room[:256, :512].nan_to_num(9.0, 8.0, -8.0), want.nan_to_num(9.0, 8.0, -8.0))
    assert bool((room[256] == 7).all()) and bool((room[:, 512:] == 7).all())


# ------------------------------------------------------------------ norm and activation
def _check_rows(rows, y, slack):
    """Codes and bytes for float64 values y that the kernel knows to a relative ``slack``: the byte is y's own, or that of a largest
    magnitude ``slack`` away; each value lies within half a step of y (the step of e4m3 at it, 2^-9 at least)."""
    b = rows.scales
    assert bool(((b == U.bytes_of(y * (1 + slack), 448.0)) | (b == U.bytes_of(y * (1 - slack), 448.0))).all())
    s = U.power(b).repeat_interleave(32, 1)
    v, got = y / s, rows.codes.float().double()
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    assert bool(((got - v).abs() <= step / 2 * (1 + 1e-9) + v.abs() * slack).all())


@pytest.mark.parametrize("m,d", [(1, 32), (3, 96), (2, 2048), (5, 2080), (3, 4096), (2, 5120), (3, 8192), (2, 8224), (1, 16416), (2, 32768), (1, 32800)])
@pytest.mark.parametrize("form", ["plain", "bf16", "f32 bias", "planes", "bias", "stream"])
def test_norm_into_8_bits(m, d, form):
    x = _randn(m, d, key=(1,)) * 2
    w = 1 + 0.1 * _randn(d, key=(2,))
    bias = 0.1 * _randn(d, key=(3,)) if "bias" in form else None
    delta = None
    if form in ("bf16", "stream"):
        delta = _randn(m, d, key=(4,)).bfloat16()
    elif form == "f32 bias":
        delta = _randn(m, d, key=(5,))
    elif form == "planes":
        delta = _randn(3, m, d, key=(6,))
    v = x.clone()
    for t in ([] if delta is None else [delta] if delta.dim() == 2 else list(delta)):
        v = v + t.float()
    if bias is not None:
        v = v + bias
    before = x.clone()
    out = kernels.Mx8.empty(m, d, DEV)
    stream = torch.empty_like(x) if form == "stream" else None
    kernels.add_rmsnorm_mx8(x, w, 1e-5, out, delta, bias, stream)
    assert torch.equal(x, before if form in ("plain", "stream") else v)      # one float32 addition after the other
    if stream is not None:
        assert torch.equal(stream, v)
    y = x.double() if form in ("plain", "stream") else before.double()         # (x holds the sum by now)
    for t in ([] if delta is None else [delta] if delta.dim() == 2 else list(delta)):
        y = y + t.double()
    if bias is not None:
        y = y + bias.double()
    if d > 32768:                                   # the stream is read again
        y = v.double()
    y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-5) * w.double()
    # 64 bits up to the one rounding: 30 of 2^-53 for the sum, the root and the products, and a root from 22 bits on (an error e
    # leaves 1.5 e^2)
    _check_rows(out, y, 2.0 ** -42)


def test_norm_of_more_rows_than_a_launch_has_threads_for():
    """2^24 rows have 256 threads each, 2^32 in all: the first and the last rows, and those on both sides of a border of 2^21 rows."""
    m, d = 2 ** 24 + 3, 32
    x = torch.empty(m, d, device=DEV).normal_(generator=_gen(22))
    delta = torch.empty(2, m, d, device=DEV, dtype=torch.bfloat16).normal_(generator=_gen(23))
    w = 1 + 0.1 * _randn(d, key=(2,))
    out, stream = kernels.Mx8.empty(m, d, DEV), torch.empty_like(x)
    kernels.add_rmsnorm_mx8(x, w, 1e-5, out, delta, stream=stream)
    assert torch.equal(stream, x + delta[0].float() + delta[1].float())
    for at in (0, 2 ** 21 - 2, 7 * 2 ** 21 - 1, 2 ** 24 - 3):
        part = slice(at, at + 6)
        y = x[part].double() + delta[0, part].double() + delta[1, part].double()
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-5) * w.double()
        _check_rows(kernels.Mx8(out.codes[part], out.scales[part]), y, 2.0 ** -42)
    del x, delta, out, stream
    torch.cuda.empty_cache()


def test_norm_of_rows_that_hold_what_is_not_finite():
    x = _randn(4, 2080)
    x[1, 40], x[2, 70] = float("nan"), float("inf")
    x[3] = 0.0
    out = kernels.add_rmsnorm_mx8(x, torch.ones(2080, device=DEV), 1e-5, kernels.Mx8.empty(4, 2080, DEV))
    got = U.values8(out.codes, out.scales)
    assert bool(got[0].isfinite().all()) and bool(got[1].isnan().all()) and bool((got[3] == 0).all())
    want = x[2].double() * 0.0                                       # over an infinite root: 0, and NaN for the infinity
    assert bool(got[2, 64:96].isnan().all()) and torch.equal(got[2, :64], want[:64]) and torch.equal(got[2, 96:], want[96:])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,d", [(1, 32), (5, 96), (3, 2080), (17, 14336)])
def test_gated_activation_into_8_bits(m, d, dtype):
    wide = torch.full((m, 2 * d + 16), float("nan"), device=DEV, dtype=dtype)
    gu = wide[:, 8:2 * d + 8]
    gu.copy_(2 * _randn(m, 2 * d))
    for bias in (None, 0.5 * _randn(2 * d, key=(1,))):
        out = kernels.swiglu_mx8(gu, kernels.Mx8.empty(m, d, DEV), bias)
        z = gu.double() if bias is None else (gu.float() + bias).double()
        g, u = z[:, :d], z[:, d:]
        # exponential, sum, quotient, product: some 2^-23 each
        _check_rows(out, g * torch.sigmoid(g) * u, 6 * 2.0 ** -23)


def test_gated_activation_far_out():
    """Gates whose exponential overflows are 0, gates that are large pass."""
    gu = torch.zeros(1, 64, device=DEV)
    gu[0, :4] = torch.tensor([-200.0, 200.0, -1e30, 1e30], device=DEV)
    gu[0, 32:36] = torch.tensor([3.0, 2.0, 1.0, 1.0], device=DEV)
    out = kernels.swiglu_mx8(gu, kernels.Mx8.empty(1, 32, DEV))
    got = U.values8(out.codes, out.scales)[0]
    assert got[0] == 0 and got[2] == 0 and abs(got[3] / 1e30 - 1) <= 2.0 ** -4 and bool((got[4:] == 0).all())


@pytest.mark.parametrize("far", [81.0, 200.0, -200.0, 1e30, float("inf"), float("nan")])
def test_a_gate_far_out_changes_no_other_block(far):
    """Rows of 96 values share waves: with one gate out of range in a row the other rows, and the other blocks of its own, keep their bits. The
    values lie within a unit or two of 1.0625, the middle between two codes, so that a last bit of silu moves them."""
    m, d = 1367, 96
    g = 2 * _randn(m, d, key=(21,))
    gu = torch.cat((g, (1.0625 / (g.double() * torch.sigmoid(g.double()))).float()), 1)
    gu[:, 0:d:32], gu[:, d::32] = 3.0, 100.0        # a block's largest: 286, so the scale is 1
    want = kernels.swiglu_mx8(gu, kernels.Mx8.empty(m, d, DEV))
    assert bool((want.scales == 127).all())
    odd = gu.clone()
    odd[2::5, 40] = far                             # a wave of 512 values holds five rows and a third
    got = kernels.swiglu_mx8(odd, kernels.Mx8.empty(m, d, DEV))
    same = torch.ones(m, d // 32, dtype=torch.bool, device=DEV)
    same[2::5, 1] = False
    assert torch.equal(got.scales[same], want.scales[same])
    assert torch.equal(_bits(got.codes).view(m, -1, 32)[same], _bits(want.codes).view(m, -1, 32)[same])


# ------------------------------------------------------------------ products
def _close(got, x, w, extra, glu=False, bias=None):
    """Within the result's rounding of the product in 64 bits, and float32 sums of k products: an addition is off by 2^-23 of the sum
    so far at most, and k of them with random signs by sqrt(k) times that; four times as much is allowed."""
    k = x.shape[1]
    y, size = x @ w.t(), torch.sqrt((x * x) @ (w * w).t())
    if bias is not None:
        y = y + bias.double()
    off = (4 * k ** 0.5 * 2.0 ** -23 + extra) * size
    if bias is not None:
        off = off + 2.0 ** -23 * bias.double().abs()
    if glu:
        g, u = y.chunk(2, 1)
        og, ou = off.chunk(2, 1)
        y = g * torch.sigmoid(g) * u
        off = 1.1 * og * u.abs() + ou * (g * torch.sigmoid(g)).abs() + 1.1 * og * ou + 2.0 ** -21 * y.abs()      # |silu'| <= 1.1
    half = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -24
    bad = (got.double() - y).abs() > half * y.abs() + off * (1 + half) + 1e-30
    assert not bool(bad.any()), (int(bad.sum()), float((got.double() - y).abs().max()))


ROWS = [1, 2, 3, 5, 8, 9, 15, 16, 17, 31, 33, 48, 64]
SHAPES = [(1, 32), (15, 64), (17, 96), (16, 128), (100, 160), (33, 512), (48, 544), (130, 1056), (1999, 2080), (64, 4096), (20, 14336)]


@pytest.mark.parametrize("n,k", SHAPES)
@pytest.mark.parametrize("m", ROWS)
def test_products_of_few_bfloat16_rows(m, n, k):
    w = _weights(n, k)
    wide = torch.full((m + 1, k + 24), float("nan"), device=DEV, dtype=torch.bfloat16)      # nothing beside the rows is read
    x = wide[:m, 8:k + 8]
    x.copy_(_randn(m, k))
    w64 = U.values4(w.codes, w.scales)
    for dtype in (torch.float32, torch.bfloat16):
        room = torch.full((m + 1, n + 7), 7.0, device=DEV, dtype=dtype)
        got = kernels.gemm_mx4(x, w, room[:m, 3:n + 3])
        assert bool((room[:, :3] == 7).all()) and bool((room[:, n + 3:] == 7).all()) and bool((room[m] == 7).all())
        _close(got, x.double(), w64, 0.0)


@pytest.mark.parametrize("n,k", [(1, 32), (16, 96), (17, 544), (130, 2080), (1000, 4096)])
@pytest.mark.parametrize("m", [1, 4, 7, 16, 23, 64])
def test_gated_products_of_few_bfloat16_rows(m, n, k):
    w, x = _weights(2 * n, k, 1), _randn(m, k, key=(1,)).bfloat16()
    bias = _randn(2 * n, key=(2,))
    w64 = U.values4(w.codes, w.scales)
    for b in (None, bias):
        for dtype in (torch.float32, torch.bfloat16):
            room = torch.full((m + 1, n + 7), 7.0, device=DEV, dtype=dtype)
            got = kernels.gemm_mx4(x, w, room[:m, 3:n + 3], b, swiglu=True)
            assert bool((room[:, :3] == 7).all()) and bool((room[:, n + 3:] == 7).all()) and bool((room[m] == 7).all())
            _close(got, x.double(), w64, 0.0, True, b)


# the unit that multiplies 8-bit rows keeps some 15 bits below the largest of 128 products: 2^-14 of it at most for each of them,
# of either sign, sqrt(128) of them in a call (11.3 * 2^-14), relative to the root of the sum of squares, which is no less
ALIGNED = 11.3 * 2.0 ** -14


@pytest.mark.parametrize("n,k", SHAPES)
@pytest.mark.parametrize("m", [1, 2, 5, 16, 17, 48, 64, 65, 127, 129, 257, 300])
def test_products_of_8_bit_rows(m, n, k):
    w, x = _weights(n, k, 2), _rows8(m, k, 2)
    for bias in (None, _randn(n, key=(3,))):
        room = torch.full((m + 1, n + 7), 7.0, device=DEV, dtype=torch.bfloat16)
        got = kernels.gemm_mx4(x, w, room[:m, 3:n + 3], bias)
        assert bool((room[:, :3] == 7).all()) and bool((room[:, n + 3:] == 7).all()) and bool((room[m] == 7).all())
        _close(got, U.values8(x.codes, x.scales), U.values4(w.codes, w.scales), ALIGNED, False, bias)


# tiles of every size: their rule goes by how many there are
@pytest.mark.parametrize("m,n,k", [(1021, 1376, 2080), (600, 4100, 448), (2011, 260, 1056), (4400, 144, 64), (2050, 2100, 224), (2049, 2056, 640),
                                   (4100, 4103, 160), (4097, 4104, 512), (513, 8200, 96)])
def test_products_of_many_8_bit_rows(m, n, k):
    w, x = _weights(n, k, 3), _rows8(m, k, 3)
    got = kernels.gemm_mx4(x, w, torch.empty(m, n, device=DEV, dtype=torch.bfloat16))
    _close(got, U.values8(x.codes, x.scales), U.values4(w.codes, w.scales), ALIGNED)


@pytest.mark.parametrize("m", [16, 17, 63, 64])
def test_gated_products_whose_gates_and_ups_lie_more_than_4_gb_apart(m):
    n, k = 2 ** 23 + 70, 512
    if torch.cuda.mem_get_info()[0] < 20e9:
        pytest.skip("wants 10 GB")
    w = kernels.Mx4.empty(2 * n, k, DEV)
    w.codes.random_(0, 256, generator=_gen(26))
    w.scales.random_(118, 124, generator=_gen(27))
    x, bias = _randn(m, k, key=(26,)).bfloat16(), _randn(2 * n, key=(26,))
    out = torch.full((m, n), float("nan"), device=DEV, dtype=torch.bfloat16)
    kernels.gemm_mx4(x, w, out, bias, swiglu=True)
    assert not bool(out.isnan().any())
    for at in (0, 2 ** 23 - 150, n - 200):          # (ending at n at most)
        cols = torch.cat((torch.arange(at, at + 200, device=DEV), torch.arange(n + at, n + at + 200, device=DEV)))
        _close(out[:, at:at + 200], x.double(), U.values4(w.codes[cols], w.scales[cols]), 0.0, True, bias[cols])
    del w, out
    torch.cuda.empty_cache()


# more weights than groups of 16 rows pay for, in one part of k and in several; k off a step, off a load of scales, and with more
# scales than LDS holds
@pytest.mark.parametrize("n,k", [(8209, 4096), (4100, 14336), (7001, 5152), (33000, 1056), (33000, 8224)])
@pytest.mark.parametrize("m", [18, 33, 64])
def test_products_of_bfloat16_rows_with_many_weights(m, n, k):
    w, x = _weights(n, k, 6), _randn(m, k, key=(6,)).bfloat16()
    w64, bias = U.values4(w.codes, w.scales), _randn(n, key=(6,))
    for dtype, b in ((torch.float32, bias), (torch.bfloat16, None)):
        room = torch.full((m + 1, n + 7), 7.0, device=DEV, dtype=dtype)
        got = kernels.gemm_mx4(x, w, room[:m, 3:n + 3], b)
        assert bool((room[:, :3] == 7).all()) and bool((room[:, n + 3:] == 7).all()) and bool((room[m] == 7).all())
        _close(got, x.double(), w64, 0.0, False, b)


@pytest.mark.parametrize("n,k", [(4100, 4096), (2050, 14336), (3501, 5152), (16500, 1056), (16500, 8224)])
@pytest.mark.parametrize("m", [19, 64])
def test_gated_products_of_bfloat16_rows_with_many_weights(m, n, k):
    w, x = _weights(2 * n, k, 7), _randn(m, k, key=(7,)).bfloat16()
    bias = _randn(2 * n, key=(7,))
    for dtype, b in ((torch.float32, bias), (torch.bfloat16, None)):
        room = torch.full((m + 1, n + 7), 7.0, device=DEV, dtype=dtype)
        got = kernels.gemm_mx4(x, w, room[:m, 3:n + 3], b, swiglu=True)
        assert bool((room[:, :3] == 7).all()) and bool((room[:, n + 3:] == 7).all()) and bool((room[m] == 7).all())
        _close(got, x.double(), U.values4(w.codes, w.scales), 0.0, True, b)


# as many columns as make a workgroup take 32: with a last one whose second 16 are there in part, or not at all
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("n,k", [(6157, 96), (8180, 544), (6160, 1056), (33000, 160), (4090, 2080), (28700, 4096)])
@pytest.mark.parametrize("m", [5, 8, 9, 16, 17, 30, 64])
def test_products_of_few_rows_with_many_columns(m, n, k, eight):
    w, x = _weights(n, k, 14), _rows8(m, k, 14) if eight else _randn(m, k, key=(14,)).bfloat16()
    bias = _randn(n, key=(14,))
    x64, w64 = U.values8(x.codes, x.scales) if eight else x.double(), U.values4(w.codes, w.scales)
    for dtype, b in ((torch.bfloat16, None), (torch.bfloat16 if eight else torch.float32, bias)):
        room = torch.full((m + 1, n + 7), 7.0, device=DEV, dtype=dtype)
        got = kernels.gemm_mx4(x, w, room[:m, 3:n + 3], b)
        assert bool((room[:, :3] == 7).all()) and bool((room[:, n + 3:] == 7).all()) and bool((room[m] == 7).all())
        _close(got, x64, w64, ALIGNED if eight else 0.0, False, b)


def _off(t):
    """The same values one byte behind a place on 16."""
    room = torch.zeros(t.numel() + 1, dtype=t.dtype, device=t.device)
    room[1:] = t.flatten()
    return room[1:].view(t.shape)


# scales off 16 bytes, by their rows' length or by where they start: every size of tile, with a part's scales in LDS at once or
# laid out again
@pytest.mark.parametrize("m,n,k", [(65, 128, 16416), (700, 1500, 4128), (1500, 2500, 2080), (1500, 4000, 2080), (2500, 4000, 2080),
                                   (60, 33000, 8224), (90, 200, 2048), (1500, 2500, 2048), (1500, 4000, 2048), (2500, 4000, 2048)])
def test_products_of_8_bit_rows_with_scales_off_16_bytes(m, n, k):
    w, x = _weights(n, k, 5), _rows8(m, k, 5)
    w, x = kernels.Mx4(w.codes, _off(w.scales)), kernels.Mx8(x.codes, _off(x.scales))
    got = kernels.gemm_mx4(x, w, torch.empty(m, n, device=DEV, dtype=torch.bfloat16))
    _close(got, U.values8(x.codes, x.scales), U.values4(w.codes, w.scales), ALIGNED)


@pytest.mark.parametrize("m,n,k", [(3, 70, 2048), (40, 70, 2048), (40, 9000, 2048), (40, 33000, 8704)])
def test_products_of_bfloat16_rows_with_scales_off_16_bytes(m, n, k):
    w, x = _weights(n, k, 5), _randn(m, k, key=(5,)).bfloat16()
    got = kernels.gemm_mx4(x, kernels.Mx4(w.codes, _off(w.scales)), torch.empty(m, n, device=DEV))
    _close(got, x.double(), U.values4(w.codes, w.scales), 0.0)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("m", [3, 40, 200])
def test_whole_numbers_are_exact(m, eight):
    """Small whole numbers under one scale: every sum is a whole number that both units hold, so nothing may be off by anything."""
    if not eight and m > kernels.MX4_MAX_ROWS:
        pytest.skip("bfloat16 rows go up to 64")
    n, k = 75, 736
    g = _gen(m, 5)
    w = torch.randint(-1, 2, (n, k), generator=g, device=DEV).float()
    w[:, ::32] = 6.0                                    # the scale of every block is 1
    x = torch.randint(-3, 4, (m, k), generator=g, device=DEV).float()
    w4 = kernels.mx4_pack(w, kernels.Mx4.empty(n, k, DEV))
    assert torch.equal(U.values4(w4.codes, w4.scales), w.double())
    if eight:
        x8 = kernels.mx8_pack(x, kernels.Mx8.empty(m, k, DEV))
        assert torch.equal(U.values8(x8.codes, x8.scales), x.double())
        got = kernels.gemm_mx4(x8, w4, torch.empty(m, n, device=DEV, dtype=torch.bfloat16))
        assert torch.equal(got, (x.double() @ w.double().t()).bfloat16())
    else:
        got = kernels.gemm_mx4(x.bfloat16(), w4, torch.empty(m, n, device=DEV))
        assert torch.equal(got.double(), x.double() @ w.double().t())


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("m", [5, 30, 150])
def test_what_is_not_finite_stays_in_its_row_and_column(m, eight):
    if not eight and m > kernels.MX4_MAX_ROWS:
        pytest.skip("bfloat16 rows go up to 64")
    n, k = 70, 1056
    w, x = _weights(n, k, 4), _randn(m, k, key=(4,))
    x[2, 1050], x[4, 0] = float("nan"), float("inf")
    w.scales[9, 32], w.scales[66, 0] = 255, 255
    a = kernels.mx8_pack(x, kernels.Mx8.empty(m, k, DEV)) if eight else x.bfloat16()
    got = kernels.gemm_mx4(a, w, torch.empty(m, n, device=DEV, dtype=torch.bfloat16))
    odd = torch.zeros(m, n, dtype=torch.bool, device=DEV)
    odd[2], odd[4], odd[:, 9], odd[:, 66] = True, True, True, True
    assert bool((got.isfinite() == ~odd).all())


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("m", [1, 20, 100])
def test_scales_at_the_ends_of_their_range(m, eight):
    """Blocks of the smallest and the largest scale against rows that bring the products back to ordinary numbers."""
    if not eight and m > kernels.MX4_MAX_ROWS:
        pytest.skip("bfloat16 rows go up to 64")
    n, k = 33, 64
    g = _gen(m, 9)
    codes = torch.randint(0, 256, (n, k // 2), generator=g, device=DEV, dtype=torch.int32).to(torch.uint8)
    for wb, e in ((1, 100), (3, 60), (253, -100), (250, -60)):
        w = kernels.Mx4(codes, torch.full((n, 2), wb, dtype=torch.uint8, device=DEV))
        x = torch.randn(m, k, generator=g, device=DEV) * 2.0 ** e
        a = kernels.mx8_pack(x, kernels.Mx8.empty(m, k, DEV)) if eight else x.bfloat16()
        got = kernels.gemm_mx4(a, w, torch.empty(m, n, device=DEV, dtype=torch.bfloat16))
        w64 = U.values4(w.codes, w.scales)
        # under the byte 253 a 6 is 6 * 2^126 = 1.5 * 2^128: no number of bfloat16, which is what a weight meets bfloat16 rows as. It
        # is an infinity there, and so is, or NaN, what it takes part in
        over = (w64.abs() >= 2.0 ** 128).any(1) & (not eight)
        assert bool(over.any()) == (wb == 253 and not eight) and not bool(got[:, over].isfinite().any())
        _close(got[:, ~over], U.values8(a.codes, a.scales) if eight else a.double(), w64[~over], ALIGNED if eight else 0.0)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("n,k", [(33, 64), (33, 1056), (9000, 2048)])
@pytest.mark.parametrize("m", [1, 8, 20, 40, 64, 100])
def test_products_under_the_smallest_and_the_largest_scale(m, n, k, eight):
    """The scale bytes 0, whose power of two is no normal float32, and 254, in every kernel; under 254 codes of less than 2, as bfloat16 holds
    nothing of 2^128 and more."""
    if not eight and m > kernels.MX4_MAX_ROWS:
        pytest.skip("bfloat16 rows go up to 64")
    g = _gen(m, n, k)
    small = torch.tensor([c for c in range(16) if c % 8 < 4], dtype=torch.uint8, device=DEV)         # 0, 0.5, 1, 1.5 and their negatives
    for byte, e in ((0, 100), (254, -100)):
        half = [small[torch.randint(0, 8, (n, k // 2), generator=g, device=DEV)] if byte else
                torch.randint(0, 16, (n, k // 2), generator=g, device=DEV, dtype=torch.uint8) for _ in range(2)]
        w = kernels.Mx4(half[0] | half[1] << 4, torch.full((n, k // 32), byte, dtype=torch.uint8, device=DEV))
        x = torch.randn(m, k, generator=g, device=DEV) * 2.0 ** e
        a = kernels.mx8_pack(x, kernels.Mx8.empty(m, k, DEV)) if eight else x.bfloat16()
        got = kernels.gemm_mx4(a, w, torch.empty(m, n, device=DEV, dtype=torch.bfloat16))
        assert bool((got != 0).any()) and bool(got.isfinite().all())
        _close(got, U.values8(a.codes, a.scales) if eight else a.double(), U.values4(w.codes, w.scales), ALIGNED if eight else 0.0)


def test_chain_captured_replayed_and_on_another_stream():
    """Norm, product, activation, product on 8-bit rows, and the gated product on bfloat16 rows: eager, recorded and replayed between other
    work, and on a stream of its own; every time the same bits."""
    m, d, di = 7, 544, 1056
    x, weight = _randn(m, d), 1 + 0.1 * _randn(d, key=(1,))
    wgu, wd = _weights(2 * di, d, 5), _weights(d, di, 6)
    h, act = kernels.Mx8.empty(m, d, DEV), kernels.Mx8.empty(m, di, DEV)
    gu = torch.empty(m, 2 * di, device=DEV, dtype=torch.bfloat16)
    out = torch.empty(m, d, device=DEV, dtype=torch.bfloat16)
    hb, side = x.bfloat16(), torch.empty(m, di, device=DEV, dtype=torch.bfloat16)

    def step():
        kernels.add_rmsnorm_mx8(x, weight, 1e-5, h)
        kernels.gemm_mx4(h, wgu, gu)
        kernels.swiglu_mx8(gu, act)
        kernels.gemm_mx4(act, wd, out)
        kernels.gemm_mx4(hb, wgu, side, swiglu=True)

    step()
    torch.cuda.synchronize()
    want = [t.clone() for t in (out, side, _bits(act.codes), act.scales)]
    # the values: what the definitions in 64 bits give from the kernels' own 8-bit rows
    _close(out, U.values8(act.codes, act.scales), U.values4(wd.codes, wd.scales), ALIGNED)
    _check_rows(act, gu.double()[:, :di] * torch.sigmoid(gu.double()[:, :di]) * gu.double()[:, di:], 6 * 2.0 ** -23)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    other = torch.cuda.Stream()
    for turn in range(4):
        for t in (out, side, act.scales, h.scales, gu):
            t.zero_()
        torch.cuda.synchronize()
        if turn == 2:
            with torch.cuda.stream(other):
                step()
        else:
            graph.replay()
        torch.cuda.synchronize()
        for t, v in zip((out, side, _bits(act.codes), act.scales), want):
            assert torch.equal(t, v), turn


@pytest.mark.parametrize("eight", [False, True])
def test_two_graphs_whose_products_are_cut_in_parts_run_at_once(eight):
    """Sums of a cut k go through scratch: two recorded products on two streams at once each keep their own."""
    m, n, k = 40, 4096, 14336
    assert kernels.gemm_mx4_scratch(eight, False, m, n, k) > 0
    runs = []
    for seed in (11, 12):
        w, x = _weights(n, k, seed), _rows8(m, k, seed) if eight else _randn(m, k, key=(seed,)).bfloat16()
        out = torch.empty(m, n, device=DEV, dtype=torch.bfloat16)
        want = kernels.gemm_mx4(x, w, out).clone()
        _close(want, U.values8(x.codes, x.scales) if eight else x.double(), U.values4(w.codes, w.scales), ALIGNED if eight else 0.0)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(20):
                kernels.gemm_mx4(x, w, out)
        runs.append((graph, torch.cuda.Stream(), out, want, w, x))
    for _ in range(3):
        for _, _, out, *_ in runs:
            out.zero_()
        torch.cuda.synchronize()
        for graph, stream, *_ in runs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, _, out, want, *_ in runs:
            assert torch.equal(out, want)


def test_more_elements_than_32_bits_count():
    m, n, k = 70000, 32768, 64
    w, x = _weights(n, k, 13), _rows8(m, k, 13)
    y = kernels.gemm_mx4(x, w, torch.empty(m, n, device=DEV, dtype=torch.bfloat16))
    for at in (0, 65535, 65536, m - 1):                       # 2^31 elements end in row 65,535
        _close(y[at:at + 1], U.values8(x.codes[at:at + 1], x.scales[at:at + 1]), U.values4(w.codes, w.scales), ALIGNED)
    rows = kernels.mx8_pack(y, kernels.Mx8.empty(m, n, DEV))
    half = kernels.swiglu_mx8(y, kernels.Mx8.empty(m, n // 2, DEV))
    for at in (65535, m - 1):
        part = slice(at, at + 1)
        v, b = U.pack8(y[part].double())
        assert torch.equal(rows.scales[part], b) and torch.equal(rows.codes[part].float().double(), v)
        gate, up = y[part].double().chunk(2, 1)
        _check_rows(kernels.Mx8(half.codes[part], half.scales[part]), gate * torch.sigmoid(gate) * up, 6 * 2.0 ** -23)
    del half
    stream = torch.empty(m, n, device=DEV).normal_(generator=_gen(13))
    last = stream[m - 1:].clone()
    weight = 1 + 0.1 * _randn(n, key=(13,))
    kernels.add_rmsnorm_mx8(stream, weight, 1e-5, rows, y)
    assert torch.equal(stream[m - 1:], last + y[m - 1:].float())
    v = last.double() + y[m - 1:].double()
    v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-5) * weight.double()
    _check_rows(kernels.Mx8(rows.codes[m - 1:], rows.scales[m - 1:]), v, 2.0 ** -42)


def test_products_of_more_rows_than_a_launch_has_threads_for():
    """2^30 rows are 2^23 tiles of 512 threads: rows on both sides of the launches' borders, every 2^26 rows, and the last."""
    m, n, k = 2 ** 30 + 70, 3, 32
    if torch.cuda.mem_get_info()[0] < 70e9:
        pytest.skip("wants 50 GB")
    w = _weights(n, k, 24)
    x = kernels.Mx8.empty(m, k, DEV)
    _bits(x.codes).random_(0, 127, generator=_gen(24))                                 # any positive value
    x.scales.random_(120, 130, generator=_gen(25))
    y = kernels.gemm_mx4(x, w, torch.full((m, n), float("nan"), device=DEV, dtype=torch.bfloat16))
    assert bool(y.isfinite().all())
    for at in (0, 2 ** 26 - 40, 5 * 2 ** 26 - 40, 2 ** 30 - 40, m - 80):
        part = slice(at, at + 80)
        _close(y[part], U.values8(x.codes[part], x.scales[part]), U.values4(w.codes, w.scales), ALIGNED)
    del x, y
    torch.cuda.empty_cache()


# ------------------------------------------------------------------ refusals
def test_nothing_to_do():
    w = _weights(40, 64)
    assert kernels.gemm_mx4(torch.empty(0, 64, device=DEV, dtype=torch.bfloat16), w, torch.empty(0, 40, device=DEV)).shape == (0, 40)
    e = kernels.Mx8.empty(0, 64, DEV)
    kernels.gemm_mx4(e, w, torch.empty(0, 40, device=DEV, dtype=torch.bfloat16))
    kernels.mx8_pack(torch.empty(0, 64, device=DEV), e)
    kernels.swiglu_mx8(torch.empty(0, 128, device=DEV), e)
    kernels.add_rmsnorm_mx8(torch.empty(0, 64, device=DEV), torch.ones(64, device=DEV), 1e-5, e, torch.empty(0, 64, device=DEV))


def test_what_is_refused():
    w, x = _weights(40, 64), _randn(3, 64).bfloat16()
    out, bf = torch.empty(3, 40, device=DEV), torch.empty(3, 40, device=DEV, dtype=torch.bfloat16)
    rows = kernels.Mx8.empty(3, 64, DEV)
    big = torch.empty(65, 64, device=DEV, dtype=torch.bfloat16)
    for call in (lambda: kernels.gemm_mx4(x.float(), w, out), lambda: kernels.gemm_mx4(x[:, :32], w, out), lambda: kernels.gemm_mx4(x, w, out[:, :39]),
                 lambda: kernels.gemm_mx4(x, w, out[:2]), lambda: kernels.gemm_mx4(x, w, out.half()), lambda: kernels.gemm_mx4(x, x, out),
                 lambda: kernels.gemm_mx4(x, w, out.t().contiguous().t()), lambda: kernels.gemm_mx4(x.t().contiguous().t(), w, out),
                 lambda: kernels.gemm_mx4(torch.empty(3, 68, device=DEV, dtype=torch.bfloat16)[:, 4:], w, out),       # off 16 bytes
                 lambda: kernels.gemm_mx4(torch.empty(3, 68, device=DEV, dtype=torch.bfloat16)[:, :64], w, out),      # rows 136 bytes apart
                 lambda: kernels.gemm_mx4(big, w, torch.empty(65, 40, device=DEV)), lambda: kernels.gemm_mx4(rows, w, out),
                 lambda: kernels.gemm_mx4(rows, w, bf, swiglu=True), lambda: kernels.gemm_mx4(x, _weights(41, 64), out, swiglu=True),
                 lambda: kernels.gemm_mx4(x, w, out, torch.zeros(39, device=DEV)), lambda: kernels.gemm_mx4(x, w, out, torch.zeros(40, device=DEV).double()),
                 lambda: kernels.gemm_mx4(x.cpu(), w, out), lambda: kernels.gemm_mx4(x, w, out.cpu()),
                 lambda: kernels.mx4_pack(x, w), lambda: kernels.mx4_pack(torch.empty(40, 64, device=DEV).half(), w),
                 lambda: kernels.mx4_unpack(w, out), lambda: kernels.mx8_pack(out, rows), lambda: kernels.mx8_pack(x[:, ::2], rows),
                 lambda: kernels.swiglu_mx8(x, rows), lambda: kernels.swiglu_mx8(torch.empty(3, 128, device=DEV), rows, torch.zeros(64, device=DEV)),
                 lambda: kernels.add_rmsnorm_mx8(x, torch.ones(64, device=DEV), 1e-5, rows),
                 lambda: kernels.add_rmsnorm_mx8(x.float(), torch.ones(63, device=DEV), 1e-5, rows),
                 lambda: kernels.add_rmsnorm_mx8(x.float(), torch.ones(64, device=DEV), 1e-5, rows, x[:2]),
                 lambda: kernels.add_rmsnorm_mx8(x.float(), torch.ones(64, device=DEV), 1e-5, rows, torch.zeros(9, 3, 64, device=DEV)),
                 lambda: kernels.add_rmsnorm_mx8(x.float(), torch.ones(64, device=DEV), 1e-5, rows, torch.zeros(0, 3, 64, device=DEV)),
                 lambda: kernels.add_rmsnorm_mx8(x.float(), torch.ones(64, device=DEV), 1e-5, rows, x, torch.zeros(8, device=DEV)),
                 lambda: kernels.add_rmsnorm_mx8(x.float(), torch.ones(64, device=DEV), 1e-5, rows, x, stream=out),
                 lambda: kernels.Mx4(w.codes, w.scales[:, :1]), lambda: kernels.Mx4(w.codes[:, :24].contiguous(), w.scales),
                 lambda: kernels.Mx4(w.codes.int(), w.scales), lambda: kernels.Mx4(w.codes[:, :16], w.scales[:, :1]),
                 lambda: kernels.Mx8(rows.codes.view(torch.uint8), rows.scales), lambda: kernels.Mx8(rows.codes, rows.scales[:2]),
                 lambda: kernels.Mx4.empty(4, 48, DEV), lambda: kernels.Mx8.empty(4, 48, DEV)):
        with pytest.raises(kernels.KernelError):
            call()


def test_more_rows_than_a_launch_counts_are_refused():
    m = 2 ** 32 + 5                                      # 5, in 32 bits
    if torch.cuda.mem_get_info()[0] < 200e9:
        pytest.skip("wants 150 GB")
    rows = kernels.Mx8.empty(m, 32, DEV)
    with pytest.raises(kernels.KernelError, match="2\\^31"):
        kernels.gemm_mx4(rows, _weights(1, 32), torch.empty(m, 1, device=DEV, dtype=torch.bfloat16))
    del rows
    torch.cuda.empty_cache()
