"""What the 4-bit and 8-bit operators refuse before they launch anything, and what a launch without a device returns; no GPU is needed."""
import pytest
import torch
from ctypes import c_float, c_int, c_longlong, c_void_p

from transformer_amd import kernels

AT = c_void_p(1 << 20)


def _gemm(lib, M=4, N=64, K=64, x=AT, codes=AT, ldx=None, ldo=None, dtype=1, glu=0, scratch=None, room=0):
    return lib.ta_gemm_mx4(None, c_int(dtype), c_int(glu), x, c_longlong(K if ldx is None else ldx), codes, AT, None, AT,
                           c_longlong(N if ldo is None else ldo), c_int(M), c_int(N), c_int(K), scratch, c_longlong(room))


def _gemm8(lib, M=4, N=64, K=64, x=AT, ldo=None, xs=AT, scratch=None, room=0):
    return lib.ta_gemm_mx4_mx8(None, x, xs, AT, AT, None, AT, c_longlong(N if ldo is None else ldo), c_int(M), c_int(N), c_int(K), scratch,
                               c_longlong(room))


def _refused(rc, name):
    lib = kernels.library()
    assert rc != 0 and lib.ta_last_error().startswith(name) and b"launch failed" not in lib.ta_last_error(), lib.ta_last_error()


def test_products_refuse_what_their_kernels_do_not_take():
    lib = kernels.library()
    off = c_void_p((1 << 20) + 8)
    for kw in (dict(K=48), dict(K=0), dict(M=-1), dict(N=0), dict(x=off), dict(codes=off), dict(ldx=68), dict(ldx=32), dict(ldo=63), dict(dtype=2),
               dict(M=65), dict(N=1 << 30, glu=1), dict(ldx=(1 << 24) + 8), dict(K=(1 << 23) + 32)):
        _refused(_gemm(lib, **kw), b"ta_gemm_mx4:")
    for kw in (dict(K=48), dict(M=-1), dict(N=0), dict(x=off), dict(ldo=63), dict(M=2147483647, N=2147483647), dict(K=(1 << 23) + 32),
               dict(M=12000, N=12000, K=2080), dict(M=12000, N=12000, K=2080, scratch=AT, room=24000 * 80 - 1),
               dict(M=12000, N=12000, K=2080, scratch=c_void_p((1 << 20) + 8), room=1 << 30),
               dict(M=12000, N=12000, K=2048, xs=c_void_p((1 << 20) + 1))):
        _refused(_gemm8(lib, **kw), b"ta_gemm_mx4_mx8:")
    assert lib.ta_mx4_max_rows() == kernels.MX4_MAX_ROWS
    # more rows: scratch for scales off 16 bytes, (rows of x in 8 bits and of the weights) * 16 bytes every 512 k, and for planes
    for K, need in ((96, 0), (512, 0), (1024, 0), (2048, 0), (2080, 24000 * 80)):
        assert kernels.gemm_mx4_scratch(True, False, 12000, 12000, K) == need
    assert kernels.gemm_mx4_scratch(True, False, 12000, 12000, 2048, False) == 24000 * 64
    for eight in (False, True):
        assert kernels.gemm_mx4_scratch(eight, False, kernels.MX_FEW_ROWS, 70, 96) == 0
        need = kernels.gemm_mx4_scratch(eight, False, 64, 4096, 14336)
        assert need and need % (64 * 4096 * 4) == 0
        call = _gemm8 if eight else _gemm
        name = b"ta_gemm_mx4_mx8:" if eight else b"ta_gemm_mx4:"
        for kw in (dict(), dict(scratch=AT, room=need - 1), dict(scratch=c_void_p((1 << 20) + 8), room=need)):
            _refused(call(lib, M=64, N=4096, K=14336, **kw), name)
    _refused(_gemm(lib, M=64, N=(1 << 23) + 1, K=512, glu=1, scratch=AT, room=1 << 62), b"ta_gemm_mx4:")     # 4 GB of gates and ups
    assert _gemm(lib, M=0) == 0 and _gemm8(lib, M=0) == 0


def test_rows_refuse_what_their_kernels_do_not_take():
    lib = kernels.library()
    off, ll = c_void_p((1 << 20) + 4), c_longlong
    for k, ld, p, dtype in ((48, 48, AT, 0), (64, 60, AT, 0), (64, 66, AT, 0), (64, 68, AT, 1), (64, 64, off, 0), (64, 64, AT, 2)):
        for name in ("ta_mx4_pack", "ta_mx8_pack"):
            _refused(getattr(lib, name)(None, c_int(dtype), p, ll(ld), AT, AT, ll(3), c_int(k)), name.encode())
        _refused(lib.ta_mx4_unpack(None, c_int(dtype), AT, AT, p, ll(ld), ll(3), c_int(k)), b"ta_mx4_unpack")
    for d, ld, p, bias, dtype in ((48, 96, AT, None, 0), (64, 124, AT, None, 0), (64, 130, AT, None, 0), (64, 132, AT, None, 1), (64, 128, off, None, 0),
                                  (64, 128, AT, off, 0), (64, 128, AT, None, 2)):
        _refused(lib.ta_swiglu_mx8(None, c_int(dtype), p, ll(ld), bias, AT, AT, ll(3), c_int(d)), b"ta_swiglu_mx8")

    def norm(n=3, d=64, planes=0, delta=None, to=AT, bias=None, x=AT, dtype=0):
        return lib.ta_add_rmsnorm_mx8(None, c_int(dtype), x, delta, c_int(planes), bias, AT, c_float(1e-5), to, AT, AT, c_int(n), c_int(d))
    for kw in (dict(d=48), dict(n=-1), dict(planes=1), dict(delta=AT), dict(planes=9, delta=AT), dict(planes=1, delta=AT, to=None), dict(bias=AT, to=None),
               dict(x=off), dict(dtype=2)):
        _refused(norm(**kw), b"ta_add_rmsnorm_mx8:")


def test_tensors_off_the_gpu_are_refused():
    codes, scales = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    for call in (lambda: kernels.Mx4(codes, scales), lambda: kernels.Mx8(torch.zeros(4, 64, dtype=torch.float8_e4m3fn), scales),
                 lambda: kernels.Mx4.empty(4, 64, "cpu"), lambda: kernels.gemm_mx4(torch.zeros(1, 64), codes, torch.zeros(1, 4)),
                 lambda: kernels.mx8_pack(torch.zeros(4, 64), None)):
        with pytest.raises(kernels.KernelError):
            call()


def test_a_launch_without_a_device_fails():
    if torch.cuda.is_available():
        pytest.skip("the operands are addresses of nothing: only where no kernel can be launched")
    lib = kernels.library()
    room = dict(scratch=AT, room=1 << 40)
    for rc, name in ((_gemm(lib), b"ta_gemm_mx4"), (_gemm(lib, glu=1, M=40, **room), b"ta_gemm_mx4"), (_gemm8(lib), b"ta_gemm_mx4_mx8"),
                     (_gemm(lib, M=64, N=4096, K=14336, **room), b"ta_gemm_mx4"), (_gemm8(lib, M=600, N=1024, K=2048, **room), b"ta_gemm_mx4_mx8")):
        assert rc != 0 and lib.ta_last_error().startswith(name), lib.ta_last_error()


def _packed(kind, n, k):
    """An ``Mx4`` or ``Mx8`` without memory."""
    t, (dtype, width) = object.__new__(kind), {kernels.Mx4: (torch.uint8, k // 2), kernels.Mx8: (torch.float8_e4m3fn, k)}[kind]
    t.codes, t.scales = torch.empty(n, width, dtype=dtype, device="meta"), torch.empty(n, k // 32, dtype=torch.uint8, device="meta")
    t.shape = (n, k)
    return t


def _bare(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("k", [2 ** 31, 2 ** 32, 2 ** 32 + 32, 2 ** 33 + 4096])
def test_a_k_beyond_a_launchs_integers_is_refused(k, monkeypatch):
    """The wrappers on tensors without memory, up to the launch, where 32 bits of such a k would pass as 0, 32 or 4,096."""
    def launch(name):
        raise AssertionError(f"{name} would be launched")
    for name, stand_in in (("_dev", lambda t, *a, **kw: t), ("_here", lambda *a: None), ("_stream", lambda: None), ("_mx", launch)):
        monkeypatch.setattr(kernels, name, stand_in)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: -1, raising=False)          # where such a tensor says that it is
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda at: 0, raising=False)
    rows, w, bf = _packed(kernels.Mx8, 1, k), _packed(kernels.Mx4, 1, k), torch.bfloat16
    for call in (lambda: kernels.mx4_pack(_bare(1, k, dtype=bf), w), lambda: kernels.mx4_unpack(w, _bare(1, k, dtype=bf)),
                 lambda: kernels.mx8_pack(_bare(1, k), rows), lambda: kernels.swiglu_mx8(_bare(1, 2 * k, dtype=bf), rows),
                 lambda: kernels.add_rmsnorm_mx8(_bare(1, k), _bare(k), 1e-5, rows),
                 lambda: kernels.add_rmsnorm_mx8(_bare(k, 32), _bare(32), 1e-5, _packed(kernels.Mx8, k, 32)),
                 lambda: kernels.add_rmsnorm_mx8(_bare(1, 32), _bare(32), 1e-5, _packed(kernels.Mx8, 1, 32), _bare(k + 1, 1, 32, dtype=bf)),
                 lambda: kernels.gemm_mx4(rows, w, _bare(1, 1, dtype=bf)), lambda: kernels.gemm_mx4(_bare(1, k, dtype=bf), w, _bare(1, 1)),
                 lambda: kernels.gemm_mx4_scratch(True, False, 64, 4096, k), lambda: kernels.gemm_mx4_scratch(True, False, k, 64, 4096),
                 lambda: kernels.gemm_mx4_scratch(True, False, 64, k, 4096)):
        with pytest.raises(kernels.KernelError, match="fewer than 2\\^31"):
            call()


def test_columns_beyond_a_launchs_threads_are_refused():
    """A launch counts its threads in 32 bits: what is beyond them is refused by name, and nothing on the way there overflows."""
    lib = kernels.library()
    for kw in (dict(M=1, N=1 << 30, K=32), dict(M=1, N=2147483647, K=32), dict(M=16, N=2147483647, K=512), dict(M=1, N=1 << 30, K=512),
               dict(M=40, N=2147483647, K=512, scratch=AT, room=1 << 62)):
        _refused(_gemm(lib, **kw), b"ta_gemm_mx4:")
        assert b"more than a launch holds" in lib.ta_last_error()
        _refused(_gemm8(lib, **kw), b"ta_gemm_mx4_mx8:")
        assert b"more than a launch holds" in lib.ta_last_error()
    for kw in (dict(M=4, N=0x3fffffff, K=512, glu=1), dict(M=1, N=0x3fffffff, K=32, glu=1)):
        _refused(_gemm(lib, **kw), b"ta_gemm_mx4:")
        assert b"more than a launch holds" in lib.ta_last_error()


def test_rows_of_several_launches_have_their_scratch_checked_before_the_first():
    """2^26 rows need none here, the 100 behind them planes."""
    lib, rows = kernels.library(), (1 << 26) + 100
    need = kernels.gemm_mx4_scratch(True, False, rows, 512, 2048)
    assert kernels.gemm_mx4_scratch(True, False, 1 << 26, 512, 2048) == 0 < need == kernels.gemm_mx4_scratch(True, False, 100, 512, 2048)
    for kw in (dict(), dict(scratch=AT, room=need - 1), dict(scratch=c_void_p((1 << 20) + 8), room=need)):
        _refused(_gemm8(lib, M=rows, N=512, K=2048, **kw), b"ta_gemm_mx4_mx8:")
        assert b"scratch" in lib.ta_last_error()


def test_what_a_launch_still_holds_goes_out():
    if torch.cuda.is_available():
        pytest.skip("the operands are addresses of nothing: only where no kernel can be launched")
    lib = kernels.library()
    for call, kw in ((_gemm, dict(M=1, N=(1 << 30) - 16, K=32)), (_gemm8, dict(M=8, N=(1 << 30) - 16, K=32)), (_gemm8, dict(M=2147483647, N=1, K=32)),
                     (_gemm8, dict(M=2147483647, N=130, K=4096, scratch=AT, room=1 << 62))):
        assert call(lib, **kw) != 0 and b"no ROCm-capable device" in lib.ta_last_error(), lib.ta_last_error()
