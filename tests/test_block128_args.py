"""What the block-scaled FP8 entry points refuse, before anything reaches a device."""
import ctypes as C

import pytest
import torch

from gpu_util import package

P = C.c_void_p(4096)            # aligned, never dereferenced: every call below is refused or has nothing to do


@pytest.fixture(scope="module")
def lib():
    return package()._capi.lib()


@pytest.fixture(scope="module")
def err():
    c = package()._capi
    return c


def text(lib):
    return lib.cf_last_error().decode()


def test_quantiser_refusals(lib, err):
    def q(x=P, ld=256, rows=4, cols=256, r8=P, ldr=256, rd=P, c8=None, ldc=0, cd=None):
        return lib.cf_fp8_quantize_block128(x, ld, rows, cols, 0, r8, ldr, rd, 2, 1, c8, ldc, cd, 256, 1, None)
    assert q(rows=0) == err.CF_OK and q(cols=0) == err.CF_OK
    for bad, words in ((dict(rows=-1), "negative"), (dict(x=None), "null input"), (dict(r8=None, rd=None), "no output"),
                       (dict(rd=None), "go together"), (dict(c8=P), "go together"), (dict(cd=P), "go together"),
                       (dict(ld=255), "input pitch"), (dict(ldr=255), "output pitch"), (dict(c8=P, cd=P, ldc=255), "output pitch"),
                       (dict(x=C.c_void_p(4097)), "misaligned"), (dict(rd=C.c_void_p(4098)), "misaligned")):
        assert q(**bad) == err.CF_ERR_INVALID_ARG, bad
        assert words in text(lib), (bad, text(lib))
    assert q(rows=0x7fffffff) == err.CF_ERR_LIMIT
    assert lib.cf_swiglu_quantize_block128(P, None, 256, 4, 256, P, 256, P, 2, 1, None, 0, None, 0, 0, None) == err.CF_ERR_INVALID_ARG
    sb = lib.cf_swiglu_backward_quantize_block128
    assert sb(P, P, 256, P, 256, 4, 192, 0, P, 384, P, 3, 1, None, 0, None, 0, 0, None) == err.CF_ERR_INVALID_ARG
    assert "multiple of 128" in text(lib)
    assert sb(P, P, 256, P, 256, 4, 256, 0, P, 511, P, 4, 1, None, 0, None, 0, 0, None) == err.CF_ERR_INVALID_ARG
    assert sb(P, P, 256, None, 256, 4, 256, 0, P, 512, P, 4, 1, None, 0, None, 0, 0, None) == err.CF_ERR_INVALID_ARG
    wq = lib.cf_fp8_quantize_block128x128
    assert wq(P, 256, 0, 0, 128, 256, P, 256, 0, P, 2, 0, None) == err.CF_OK
    assert wq(P, 255, 0, 1, 128, 256, P, 256, 0, P, 2, 0, None) == err.CF_ERR_INVALID_ARG
    assert wq(P, 256, 0, 1, 128, 256, P, 256, 0, P, 1, 0, None) == err.CF_ERR_INVALID_ARG
    assert wq(P, 256, 128, 2, 128, 256, P, 256, 128 * 256, P, 2, 2, None) == err.CF_ERR_INVALID_ARG and "overlap" in text(lib)
    assert wq(None, 256, 0, 1, 128, 256, P, 256, 0, P, 2, 0, None) == err.CF_ERR_INVALID_ARG


def test_norm_refusals(lib, err):
    def n(x=P, res=None, g=P, h=None, normed=P, out8=None, ld8=0, d=None, rows=4, H=256, eps=1e-6):
        return lib.cf_add_rmsnorm_quantize_block128(x, res, g, h, normed, None, out8, ld8, d, 2, 1, rows, H, eps, None)
    assert n(rows=0) == err.CF_OK
    for bad in (dict(rows=-1), dict(H=0), dict(eps=0.0), dict(x=None), dict(g=None), dict(normed=None), dict(res=P), dict(out8=P, ld8=256),
                dict(d=P), dict(out8=P, d=P, ld8=255), dict(x=C.c_void_p(4097))):
        assert n(**bad) == err.CF_ERR_INVALID_ARG, bad
    assert n(H=16385) == err.CF_ERR_LIMIT
    f = lib.cf_add_rmsnorm_backward_scratch_floats
    # one partial row per block, as many blocks as rows up to a fixed number
    assert f(0, 256) == 0 and f(1, 256) == 256 and f(10 ** 6, 4096) == f(10 ** 5, 4096) > 0 and f(4, 16385) == 0

    def b(dy=P, h=P, g=P, rms=P, dx=P, dg=P, scratch=P, n=1024, rows=4, H=256):
        return lib.cf_add_rmsnorm_backward(dy, h, g, rms, None, dx, dg, 0, scratch, n, rows, H, None)
    for bad in (dict(rows=-1), dict(H=0), dict(dy=None), dict(h=None), dict(g=None), dict(rms=None), dict(dx=None), dict(dx=C.c_void_p(4097))):
        assert b(**bad) == err.CF_ERR_INVALID_ARG, bad
    assert b(n=1023) == err.CF_ERR_LIMIT and b(scratch=None) == err.CF_ERR_LIMIT and b(H=16385) == err.CF_ERR_LIMIT


def test_product_refusals(lib, err):
    room = C.create_string_buffer(1 << 16)                 # stands for a context: only its status pointer is read, as null
    ctx = C.cast(room, C.c_void_p)

    def nt(ctx=ctx, M=300, N=256, K=256, A=P, lda=256, sa=P, B=P, ldb=256, sb=P, per=128, out=P, ldc=256, f32=0):
        return lib.cf_gemm_fp8_block128_nt(ctx, M, N, K, A, lda, 0, sa, 2, 1, B, ldb, sb, 2, 1, per, out, ldc, f32, 0, None)
    for bad in (dict(ctx=None), dict(M=-1), dict(K=-1), dict(A=None), dict(B=None), dict(sa=None), dict(sb=None), dict(out=None),
                dict(lda=240), dict(ldb=240), dict(ldc=255), dict(per=64), dict(out=C.c_void_p(4098), f32=1), dict(sa=C.c_void_p(4097))):
        assert nt(**bad) == err.CF_ERR_INVALID_ARG, bad
    for bad in (dict(A=C.c_void_p(4104)), dict(B=C.c_void_p(4097)), dict(lda=264), dict(ldb=257)):
        assert nt(**bad) == err.CF_ERR_UNSUPPORTED, bad
    assert nt(M=0x7fffffff) == err.CF_ERR_LIMIT
    assert nt(K=0, A=None, B=None, sa=None, sb=None, ldc=255) == err.CF_ERR_INVALID_ARG
    g = lib.cf_gemm_fp8_block128_nt_grouped

    def grouped(E=2, T=300, counts=P, offsets=P, ldb=256, N=256):
        return g(ctx, E, T, N, 256, counts, offsets, P, 256, 0, P, 2, 1, P, ldb, P, 2, 4, P, N, None)
    for bad in (dict(E=0), dict(counts=None), dict(offsets=None), dict(ldb=255), dict(T=-1)):
        assert grouped(**bad) == err.CF_ERR_INVALID_ARG, bad
    assert grouped(E=1 << 24, N=256) == err.CF_ERR_LIMIT and grouped(E=65537, N=16) == err.CF_ERR_LIMIT
    nn = lib.cf_gemm_fp8_block128_nn
    assert nn(ctx, 300, 256, 256, P, 256, 0, P, 2, 1, P, 255, P, 2, P, 256, 0, 0, None) == err.CF_ERR_INVALID_ARG
    assert nn(ctx, 300, 256, 256, P, 256, 0, P, 2, 1, P, 264, P, 2, P, 256, 0, 0, None) == err.CF_ERR_UNSUPPORTED
    dw = lib.cf_gemm_fp8_block128_dw
    assert dw(ctx, 300, 256, 256, P, 299, 0, P, 300, 1, P, 256, 0, P, 256, 1, P, 256, 1, 0, None) == err.CF_ERR_INVALID_ARG
    assert dw(ctx, 300, 256, 256, P, 300, 0, P, 300, 1, P, 256, 0, P, 256, 1, P, 256, 1, 0, None) == err.CF_ERR_UNSUPPORTED


class _Dev:
    """Stands for a device tensor of a given shape: what the wrappers look at before they pass a pointer on."""

    def __init__(self, t, device=0):
        self.t, self.index = t, device

    def get_device(self):
        return self.index

    def __getattr__(self, name):
        return getattr(self.t, name)

    def __getitem__(self, i):
        return _Dev(self.t[i])

    def data_ptr(self):
        return 4096


def dev(*shape, dtype=torch.bfloat16, of=None):
    return _Dev(torch.empty(shape, dtype=dtype) if of is None else of)


def test_wrappers_refuse_tensors_that_do_not_fit(monkeypatch):
    cfb = package()
    monkeypatch.setattr(cfb.ops, "_s", lambda: None)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    u8, f32 = torch.uint8, torch.float32
    ctx = type("Ctx", (), {"handle": P})()

    def refused(fn, *a, **k):
        with pytest.raises(cfb.CanopyError) as e:
            fn(*a, **k)
        assert e.value.code == cfb._capi.CF_ERR_INVALID_ARG

    q = cfb.fp8_quantize_block128
    x = dev(4, 256)
    refused(q, x, dev(4, 255, dtype=u8), dev(4, 2, dtype=f32))
    refused(q, x, dev(4, 256, dtype=u8), dev(4, 3, dtype=f32))
    refused(q, x, dev(4, 256, dtype=u8), dev(4, 2))
    refused(q, x, dev(4, 256, dtype=u8))
    refused(q, x)
    refused(q, dev(4, 256, dtype=f32), dev(4, 256, dtype=u8), dev(4, 2, dtype=f32))
    refused(q, dev(of=torch.empty((256, 4), dtype=torch.bfloat16).t()), dev(4, 256, dtype=u8), dev(4, 2, dtype=f32))
    refused(q, dev(of=torch.empty((1, 256), dtype=torch.bfloat16).expand(4, 256)), dev(4, 256, dtype=u8), dev(4, 2, dtype=f32))
    refused(cfb.swiglu_quantize_block128, x, dev(of=torch.empty((4, 512), dtype=torch.bfloat16)[:, :256]), dev(4, 256, dtype=u8), dev(4, 2, dtype=f32))
    refused(cfb.swiglu_backward_quantize_block128, x, x, x, dev(4, 256, dtype=u8), dev(4, 2, dtype=f32))
    refused(cfb.fp8_quantize_block128x128, x, dev(4, 256, dtype=u8), dev(2, 2, dtype=f32))
    g = dev(256)
    refused(cfb.add_rmsnorm_quantize_block128, x, dev(4, 255), g, x, None, x)
    refused(cfb.add_rmsnorm_quantize_block128, x, None, dev(255), None, None, x)
    refused(cfb.add_rmsnorm_quantize_block128, x, None, g, None, dev(3, dtype=f32), x)
    refused(cfb.add_rmsnorm_backward, x, x, g, dev(4, dtype=f32), None, dev(4, 256, dtype=f32))
    A, da = dev(300, 256, dtype=u8), dev(300, 2, dtype=f32)
    B, db = dev(256, 256, dtype=u8), dev(2, 2, dtype=f32)
    out = dev(300, 256)
    refused(cfb.gemm_fp8_block128_nt, ctx, A, dev(300, 3, dtype=f32), B, db, out)
    refused(cfb.gemm_fp8_block128_nt, ctx, A, da, B, dev(3, 2, dtype=f32), out)
    refused(cfb.gemm_fp8_block128_nt, ctx, A, da, dev(256, 128, dtype=u8), db, out)
    refused(cfb.gemm_fp8_block128_nt, ctx, A, da, B, db, dev(300, 255))
    refused(cfb.gemm_fp8_block128_nt, ctx, A, da, B, db, dev(300, 256, dtype=torch.float16))
    refused(cfb.gemm_fp8_block128_nn, ctx, A, da, B, dev(of=torch.empty((2, 2)).t()), out)
    refused(cfb.gemm_fp8_block128_dw, ctx, A, dev(3, 256, dtype=f32), dev(301, 256, dtype=u8), dev(3, 256, dtype=f32), dev(256, 256, dtype=f32))
    E8 = dev(2, 256, 256, dtype=u8)
    c = dev(2, dtype=torch.int32)
    refused(cfb.gemm_fp8_block128_nt_grouped, ctx, dev(3, dtype=torch.int32), c, A, da, E8, dev(2, 2, 2, dtype=f32), out)
    refused(cfb.gemm_fp8_block128_nt_grouped, ctx, dev(2, dtype=torch.int64), c, A, da, E8, dev(2, 2, 2, dtype=f32), out)
    refused(cfb.gemm_fp8_block128_nt_grouped, ctx, c, c, A, da, dev(of=torch.empty((2, 300, 256), dtype=u8)[:, :256]), dev(2, 2, 2, dtype=f32), out)
    refused(cfb.gemm_fp8_block128_nt_grouped, ctx, c, c, A, da, E8, dev(2, 2, 2, dtype=f32), dev(300, 256, dtype=f32))


def test_wrappers_refuse_sizes_beyond_an_int(monkeypatch):
    """Sizes and pitches cross to C as ints: 2^32 + 256 would arrive there as 256, a call that looks right."""
    cfb = package()
    monkeypatch.setattr(cfb.ops, "_s", lambda: None)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    ctx = type("Ctx", (), {"handle": P})()
    u8, f32, bf16, far = torch.uint8, torch.float32, torch.bfloat16, (1 << 32) + 256

    def meta(*shape, dtype=bf16):
        return torch.empty(shape, dtype=dtype, device="meta")

    def big(*shape, dtype=bf16):
        return dev(of=meta(*shape, dtype=dtype))

    def wide(rows, cols, dtype=bf16):
        return dev(of=meta(rows, far, dtype=dtype)[:, :cols])

    c8, rd, d = dev(4, 256, dtype=u8), dev(4, 2, dtype=f32), dev(1, 2, dtype=f32)
    x, out, g = dev(4, 256), dev(4, 4), dev(256)
    E8, ed = big(far, 1, 128, dtype=u8), big(far, 1, 1, dtype=f32)
    i = big(far, dtype=torch.int32)
    for fn, args in ((cfb.fp8_quantize_block128, (wide(4, 256), c8, rd)),
                     (cfb.fp8_quantize_block128, (x, wide(4, 256, u8), rd)),
                     (cfb.fp8_quantize_block128, (x, None, None, wide(4, 256, u8), dev(1, 256, dtype=f32))),
                     (cfb.fp8_quantize_block128, (big(1, far), big(1, far, dtype=u8), big(1, far // 128, dtype=f32))),
                     (cfb.fp8_quantize_block128, (big(far, 1), big(far, 1, dtype=u8), big(far, 1, dtype=f32))),
                     (cfb.fp8_quantize_block128x128, (wide(4, 256), c8, d)),
                     (cfb.fp8_quantize_block128x128, (big(far, 1, 1), big(far, 1, 1, dtype=u8), ed)),
                     (cfb.add_rmsnorm_quantize_block128, (big(far, 256), None, g, None, None, big(far, 256))),
                     (cfb.add_rmsnorm_backward, (big(far, 256), big(far, 256), g, big(far, dtype=f32), None, big(far, 256))),
                     (cfb.gemm_fp8_block128_nt, (ctx, wide(4, 256, u8), rd, c8, d, out)),
                     (cfb.gemm_fp8_block128_nt, (ctx, c8, rd, c8, d, wide(4, 4))),
                     (cfb.gemm_fp8_block128_dw, (ctx, c8, dev(1, 256, dtype=f32), wide(4, 4, u8), dev(1, 4, dtype=f32), dev(256, 4, dtype=f32))),
                     (cfb.gemm_fp8_block128_nt_grouped, (ctx, i, i, dev(4, 128, dtype=u8), dev(4, 1, dtype=f32), E8, ed, dev(4, 1))),
                     (cfb.gemm_fp8_block128_nt_grouped, (ctx, dev(0, dtype=torch.int32), dev(0, dtype=torch.int32), dev(4, 128, dtype=u8),
                                                         dev(4, 1, dtype=f32), dev(0, 4, 128, dtype=u8), dev(0, 1, 1, dtype=f32), out))):
        with pytest.raises(cfb.CanopyError) as e:
            fn(*args)
        assert e.value.code == cfb._capi.CF_ERR_INVALID_ARG, fn.__name__


def test_wrappers_refuse_tensors_of_another_device(monkeypatch):
    """The call goes to the current device's stream: a tensor on the CPU or on another GPU is refused, by every operator."""
    cfb = package()
    monkeypatch.setattr(cfb.ops, "_s", lambda: None)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    ctx = type("Ctx", (), {"handle": P})()
    u8, f32 = torch.uint8, torch.float32
    x, g, c8, d, out = dev(256, 256), dev(256), dev(256, 256, dtype=u8), dev(2, 2, dtype=f32), dev(256, 256)
    rd, cd, v, i = dev(256, 2, dtype=f32), dev(2, 256, dtype=f32), dev(256, dtype=f32), dev(1, dtype=torch.int32)
    W, e8, ed = dev(2, 256, 256), dev(1, 256, 256, dtype=u8), dev(1, 2, 2, dtype=f32)
    rd2, c82 = dev(256, 4, dtype=f32), dev(256, 512, dtype=u8)
    scratch = dev(1 << 20, dtype=f32)
    calls = ((cfb.fp8_quantize_block128, (x, c8, rd, c8, cd)), (cfb.swiglu_quantize_block128, (x, x, c8, rd, c8, cd)),
             (cfb.swiglu_backward_quantize_block128, (x, x, x, c82, rd2)), (cfb.fp8_quantize_block128x128, (x, c8, d)),
             (cfb.add_rmsnorm_quantize_block128, (x, x, g, x, v, x, c8, rd)), (cfb.add_rmsnorm_backward, (x, x, g, v, x, x, v, scratch)),
             (cfb.gemm_fp8_block128_nt, (ctx, c8, rd, c8, d, out)), (cfb.gemm_fp8_block128_nt_grouped, (ctx, i, i, c8, rd, e8, ed, out)),
             (cfb.gemm_fp8_block128_nn, (ctx, c8, rd, c8, d, out)), (cfb.gemm_fp8_block128_dw, (ctx, c8, cd, c8, cd, out)))
    for fn, args in calls:
        for k, a in enumerate(args):
            if isinstance(a, _Dev):
                for other in (-1, 1):
                    moved = args[:k] + (_Dev(a.t, other),) + args[k + 1:]
                    with pytest.raises(cfb.CanopyError) as e:
                        fn(*moved)
                    assert e.value.code == cfb._capi.CF_ERR_INVALID_ARG and "device" in str(e.value), (fn.__name__, k)


def test_grouped_product_of_single_rows_refuses_a_pitch_beyond_an_int(monkeypatch):
    """Experts of one row each lie one pitch apart: 2^32 + 256 would reach the library as 256, the rows of other experts."""
    cfb = package()
    monkeypatch.setattr(cfb.ops, "_s", lambda: None)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    passed = []
    fake = type("Lib", (), {"cf_gemm_fp8_block128_nt_grouped": lambda self, *a: passed.append(a) or 0})()
    monkeypatch.setattr(cfb.ops, "_L", lambda: fake)
    ctx = type("Ctx", (), {"handle": P})()
    u8, f32 = torch.uint8, torch.float32
    i, A, da, db, out = dev(2, dtype=torch.int32), dev(4, 128, dtype=u8), dev(4, 1, dtype=f32), dev(2, 1, 1, dtype=f32), dev(4, 1)
    for pitch, fits in ((256, True), ((1 << 31) - 16, True), (1 << 31, False), ((1 << 32) + 256, False)):
        B8 = dev(of=torch.empty((2, 1, pitch), dtype=u8, device="meta")[..., :128])
        if fits:
            cfb.gemm_fp8_block128_nt_grouped(ctx, i, i, A, da, B8, db, out)
            assert passed.pop()[14] == pitch                 # ldb
        else:
            with pytest.raises(cfb.CanopyError) as e:
                cfb.gemm_fp8_block128_nt_grouped(ctx, i, i, A, da, B8, db, out)
            assert e.value.code == cfb._capi.CF_ERR_INVALID_ARG and not passed


def test_feed_forward_block_after_a_refused_call(monkeypatch):
    """A call of too many rows changes nothing: backward() still differentiates the call before it. A call that is refused on its
    way has overwritten what the call before it kept: nothing is left to differentiate."""
    cfb = package()
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    done = []
    for name in ("add_rmsnorm_quantize_block128", "gemm_fp8_block128_nt", "gemm_fp8_block128_nn", "gemm_fp8_block128_dw", "swiglu_quantize_block128",
                 "swiglu_backward_quantize_block128", "add_rmsnorm_backward", "fp8_quantize_block128", "fp8_quantize_block128x128"):
        monkeypatch.setattr(cfb.ops, name, lambda *a, _n=name, **k: done.append((_n, a)))
    H, F = 256, 128
    ctx = type("Ctx", (), {"handle": P})()
    block = cfb.FfnSwigluFp8Block128(ctx, 4, H, F, train=True, device="cpu")

    def bf16(*shape):
        return torch.empty(shape, dtype=torch.bfloat16)

    wgu, wd = cfb.Fp8Block128Weight(bf16(2 * F, H)), cfb.Fp8Block128Weight(bf16(H, F))
    gain, dw, dd, dg = bf16(H), torch.empty(2 * F, H), torch.empty(H, F), torch.empty(H)

    def backward(n):
        done.clear()
        block.backward(bf16(n, H), None, gain, wgu, wd, bf16(n, H), dw, dd, dg)
        return [a[1].shape[0] for name, a in done if name == "gemm_fp8_block128_nn"]

    def refused(fn):
        with pytest.raises(cfb.CanopyError) as e:
            fn()
        assert e.value.code == cfb._capi.CF_ERR_INVALID_ARG

    refused(lambda: backward(3))                             # nothing has run
    block.forward(bf16(3, H), None, gain, wgu, wd, bf16(3, H))
    assert backward(3) == [3, 3]
    refused(lambda: block.forward(bf16(5, H), None, gain, wgu, wd, bf16(5, H)))
    assert backward(3) == [3, 3]
    monkeypatch.setattr(cfb.ops, "swiglu_quantize_block128", lambda *a: cfb.ops._refuse("on its way"))
    refused(lambda: block.forward(bf16(2, H), None, gain, wgu, wd, bf16(2, H)))
    refused(lambda: backward(2))
    refused(lambda: backward(3))
