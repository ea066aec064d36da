"""Block-scaled FP8 operators (one scale per 128 values) against their definitions in 64 bits.

Tolerances count roundings: a rounding to a type is off by at most eps / 2 of the value (bf16 2^-8, E4M3 2^-4, E5M2 2^-3, and
half the smallest subnormal of the FP8 types below their normal range), and every fp32 operation by 2^-24 of its result."""
import numpy as np
import pytest
import torch

from gpu_util import package

pytestmark = pytest.mark.gpu

G = 128
FMAX = {False: 448.0, True: 57344.0}
TYPE = {False: torch.float8_e4m3fn, True: torch.float8_e5m2}
HALF = {False: 2.0 ** -4, True: 2.0 ** -3}          # half a step, relative
TINY = {False: 2.0 ** -10, True: 2.0 ** -17}        # half the smallest subnormal
U = 2.0 ** -24                                       # fp32 rounding


@pytest.fixture(scope="module")
def cfb():
    return package()


@pytest.fixture(scope="module")
def ctx(cfb):
    c = cfb.Fp8Ctx()
    yield c
    c.poll_status()
    c.close()


def cdiv(a, b):
    return -(-a // b)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(shape, seed, std=1.0):
    return (torch.randn(shape, generator=gen(seed), device="cuda") * std).to(torch.bfloat16)


def pitched(rows, cols, dtype, pad, offset=0, fill=0x5a):
    """A [rows, cols] view with `pad` extra elements per row, `offset` elements into its buffer, and the buffer's bytes."""
    size = torch.empty((), dtype=dtype).element_size()
    raw = torch.full(((rows * (cols + pad) + offset + 64) * size,), fill, dtype=torch.uint8, device="cuda")
    flat = raw.view(dtype)[offset:]
    return flat[: rows * (cols + pad)].view(rows, cols + pad)[:, :cols], raw


def decode(codes, e5m2):
    return codes.contiguous().view(TYPE[e5m2]).double()


def groups64(v, dim):
    """max |v| of groups of 128 along dim, floored, in v's shape (spread over the group) and per group."""
    n = v.shape[dim]
    per = torch.stack([p.abs().amax(dim) for p in torch.split(v, G, dim)], dim).clamp(min=1e-12)
    return per.repeat_interleave(G, dim).narrow(dim, 0, n), per


def check_groups(codes, descale, v, dim, e5m2, slack):
    """codes * descale is v up to one rounding to the type, descale is amax / FMAX; slack: relative fp32 error of v itself."""
    a, per = groups64(v, dim)
    assert (descale.double() - per / FMAX[e5m2]).abs().le((slack + 2 * U) * per / FMAX[e5m2]).all()
    want = v / a * FMAX[e5m2]
    err = (decode(codes, e5m2) - want).abs()
    # v's own error and three fp32 operations (the scale's division, the product, the amax) move the value before it is rounded
    bound = torch.maximum(want.abs() * HALF[e5m2], torch.full_like(want, TINY[e5m2])) * (1 + 2.0 ** -10) + want.abs() * (slack + 4 * U)
    assert err.le(bound).all(), float((err - bound).max())


def nearest64(v, e5m2):
    """Codes of the 64-bit values: round to nearest, ties to even, from the format's definition."""
    mant, low = (2, -14) if e5m2 else (3, -6)
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), torch.clamp(e - 1, min=low) - mant)
    return torch.clamp(torch.round(v / step) * step, -FMAX[e5m2], FMAX[e5m2]).to(TYPE[e5m2]).view(torch.uint8)


def plain_codes(x, dim, e5m2):
    """Codes and descales of a bf16 matrix from the 64-bit quotients. (v * FMAX is exact in 64 bits and the quotient of an 11-bit
    and an 8-bit number is either representable or further than 2^-20 from every code's border: no double rounding.)"""
    v = x.double()
    a, per = groups64(v, dim)
    a, per = a.float().double(), per.float().double()
    return nearest64(v * FMAX[e5m2] / a, e5m2), (per / FMAX[e5m2]).float()


# ---------------------------------------------------------------- quantiser
SHAPES = [(1, 1), (1, 4096), (3, 127), (128, 128), (129, 257), (130, 136), (300, 1000), (1027, 513), (16, 8), (2048, 1024)]


@pytest.mark.parametrize("e5m2", [False, True])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantise_rows_and_columns_bit_exact(cfb, rows, cols, e5m2):
    x = normal((rows, cols), rows * 7 + cols)
    if cols > 4:
        x[0, 3] = 30.0
    x[rows // 2] = 0.0                                   # a row of zeros: the floor of the amax
    for which in ("row", "col", "both"):
        row8 = torch.empty((rows, cols), dtype=torch.uint8, device="cuda") if which != "col" else None
        rd = torch.empty((rows, cdiv(cols, G)), device="cuda") if which != "col" else None
        col8 = torch.empty((rows, cols), dtype=torch.uint8, device="cuda") if which != "row" else None
        cd = torch.empty((cdiv(rows, G), cols), device="cuda") if which != "row" else None
        cfb.fp8_quantize_block128(x, row8, rd, col8, cd, is_e5m2=e5m2)
        if which != "col":
            q, d = plain_codes(x, 1, e5m2)
            assert torch.equal(row8, q) and torch.equal(rd, d), which
        if which != "row":
            q, d = plain_codes(x, 0, e5m2)
            assert torch.equal(col8, q) and torch.equal(cd, d), which
        if which == "both":
            check_groups(row8, rd, x.double(), 1, e5m2, 0.0)
            check_groups(col8, cd, x.double(), 0, e5m2, 0.0)


@pytest.mark.parametrize("pad,offset", [(0, 1), (1, 0), (8, 8), (3, 5)])
def test_quantise_pitches_and_alignments_leave_the_rest(cfb, pad, offset):
    rows, cols = 141, 261
    x, _ = pitched(rows, cols, torch.bfloat16, pad, offset)
    x.copy_(normal((rows, cols), 3))
    row8, raw_r = pitched(rows, cols, torch.uint8, pad, offset)
    col8, raw_c = pitched(rows, cols, torch.uint8, pad, offset)
    rd = cfb.block128_row_descale(rows, cols)            # [groups, rows] in memory
    cd = torch.full((cols, cdiv(rows, G)), -1.0, device="cuda").t()
    cfb.fp8_quantize_block128(x, row8, rd, col8, cd)
    q, d = plain_codes(x, 1, False)
    assert torch.equal(row8, q) and torch.equal(rd, d)
    q, d = plain_codes(x, 0, False)
    assert torch.equal(col8, q) and torch.equal(cd, d)
    for view, raw in ((row8, raw_r), (col8, raw_c)):     # nothing outside the matrix was written
        view.fill_(0x5a)
        assert raw.eq(0x5a).all()


def test_quantise_infinities_and_nan(cfb):
    x = normal((4, 256), 5)
    x[0, 5] = float("inf")
    x[1, 7] = float("nan")
    x[2, 200] = float("-inf")
    row8 = torch.empty((4, 256), dtype=torch.uint8, device="cuda")
    rd = torch.empty((4, 2), device="cuda")
    cfb.fp8_quantize_block128(x, row8, rd)
    v = decode(row8, False) * rd.double().repeat_interleave(G, 1)
    assert torch.isinf(rd[0, 0]) and v[0, :128].isnan().all()
    assert v[1, 7].isnan() and torch.isfinite(v[1, :7]).all() and torch.isfinite(rd[1]).all()
    assert torch.isfinite(v[2, :128]).all() and v[2, 128:].isnan().all()
    clean = normal((4, 256), 5)
    q, d = plain_codes(clean, 1, False)
    assert torch.equal(row8[3], q[3]) and torch.equal(rd[3], d[3])


@pytest.mark.parametrize("e5m2", [False, True])
@pytest.mark.parametrize("both", [False, True])
def test_quantise_columns_infinities_and_nan(cfb, e5m2, both):
    x = normal((200, 136), 6)
    x[3, 5], x[150, 7], x[60, 130], x[:128, 9] = float("inf"), float("-inf"), float("nan"), float("nan")
    col8 = torch.empty((200, 136), dtype=torch.uint8, device="cuda")
    cd = torch.empty((2, 136), device="cuda")
    row8, rd = (torch.empty_like(col8), torch.empty((200, 2), device="cuda")) if both else (None, None)
    cfb.fp8_quantize_block128(x, row8, rd, col8, cd, is_e5m2=e5m2)
    clean = torch.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0)
    q, d = plain_codes(clean, 0, e5m2)
    holds = torch.zeros((2, 136), dtype=torch.bool, device="cuda")
    holds[0, 5] = holds[1, 7] = True
    assert torch.isinf(cd[holds]).all() and torch.equal(cd[~holds], d[~holds])
    v = decode(col8, e5m2)
    assert (v * cd.double().repeat_interleave(G, 0)[:200])[holds.repeat_interleave(G, 0)[:200]].isnan().all()
    rest = ~(holds.repeat_interleave(G, 0)[:200] | x.isnan())
    assert torch.equal(col8[rest], q[rest]) and v[x.isnan()].isnan().all()


def test_quantise_weight_blocks_infinities_and_nan(cfb):
    w = normal((260, 300), 12, 0.02)
    w[5, 200], w[140, 3], w[256:, 256:] = float("-inf"), float("nan"), float("nan")
    w8, d = torch.empty((260, 300), dtype=torch.uint8, device="cuda"), torch.empty((3, 3), device="cuda")
    cfb.fp8_quantize_block128x128(w, w8, d)
    v = decode(w8, False) * d.double().repeat_interleave(G, 0)[:260].repeat_interleave(G, 1)[:, :300]
    assert torch.isinf(d[0, 1]) and v[:128, 128:256].isnan().all() and int(torch.isinf(d).sum()) == 1
    assert v[140, 3].isnan() and int(v[128:256, :128].isnan().sum()) == 1
    assert v[256:, 256:].isnan().all() and d[2, 2] == (torch.tensor(1e-12).double() / 448.0).float()
    clean = torch.nan_to_num(w, nan=0.0, posinf=0.0, neginf=0.0)
    c8, cd = torch.empty_like(w8), torch.empty_like(d)
    cfb.fp8_quantize_block128x128(clean, c8, cd)
    d[0, 1] = cd[0, 1]
    assert torch.equal(d, cd)
    rest = torch.isfinite(w)
    rest[:128, 128:256] = False
    assert torch.equal(w8[rest], c8[rest])


@pytest.mark.parametrize("shape", [(1, 1), (128, 128), (130, 260), (256, 1000), (5, 129), (3, 130, 140), (2, 128, 256), (4, 1, 16)])
def test_quantise_weight_blocks_bit_exact(cfb, shape):
    w = normal(shape, 11, 0.02)
    w8 = torch.empty(shape, dtype=torch.uint8, device="cuda")
    d = torch.empty((*shape[:-2], cdiv(shape[-2], G), cdiv(shape[-1], G)), device="cuda")
    cfb.fp8_quantize_block128x128(w, w8, d)
    for i in range(cdiv(shape[-2], G)):
        for j in range(cdiv(shape[-1], G)):
            part = w[..., i * G:(i + 1) * G, j * G:(j + 1) * G].double()
            a = part.abs().amax((-2, -1), keepdim=True).clamp(min=1e-12)
            q = nearest64(part * 448.0 / a, False)
            assert torch.equal(w8[..., i * G:(i + 1) * G, j * G:(j + 1) * G], q)
            assert torch.equal(d[..., i, j], (a.double() / 448.0).float()[..., 0, 0])


# expf is off by 2 units (2^-23 each), the sigmoid's sum and division by one rounding each, then two products
SWIGLU_SLACK = 8 * 2.0 ** -23


@pytest.mark.parametrize("rows,cols", [(1, 14336), (5, 130), (129, 384), (300, 1001)])
def test_swiglu_quantise(cfb, rows, cols):
    gu = normal((rows, 2 * cols), 21, 2.0)
    gate, up = gu[:, :cols], gu[:, cols:]
    row8 = torch.empty((rows, cols), dtype=torch.uint8, device="cuda")
    rd = cfb.block128_row_descale(rows, cols)
    col8 = torch.empty_like(row8)
    cd = torch.empty((cdiv(rows, G), cols), device="cuda")
    cfb.swiglu_quantize_block128(gate, up, row8, rd, col8, cd)
    v = gate.double() * torch.sigmoid(gate.double()) * up.double()
    check_groups(row8, rd, v, 1, False, SWIGLU_SLACK)
    check_groups(col8, cd, v, 0, False, SWIGLU_SLACK)
    only = torch.empty_like(row8)
    cfb.swiglu_quantize_block128(gate, up, only, rd.clone())
    assert torch.equal(only, row8)


FAR = [60.0, -60.0, -80.0, -85.0, -87.0, -88.0, 100.0, -100.0, 1e4, -1e4, 1e30, -1e30, 3e38, -3e38]
# 1 / (1 + exp(-g)) is taken as zero where it is below the smallest normal number, 2^-126, that is for g below -87.3: there |silu| <
# 87.4 * 2^-126 < 2^-119, and each gradient's factor is smaller than that
FLUSHED = 2.0 ** -119


def test_swiglu_far_gates(cfb):
    """Gates far from zero, one in each group of 128 columns, in forward and gradient: right to the bounds of the operator's
    arithmetic, a vanishing silu times a huge up included."""
    n = len(FAR)
    for u in (1.0, -3.0, 1e30):
        gate = torch.zeros((n, G), dtype=torch.bfloat16, device="cuda")
        gate[:, 7] = torch.tensor(FAR, device="cuda").to(torch.bfloat16)
        up, dh = torch.zeros_like(gate), torch.zeros_like(gate)
        up[:, 7], dh[:, 7] = u, 0.5
        g, uu, d = (t[:, 7].double() for t in (gate, up, dh))
        s, rest = torch.sigmoid(g), torch.sigmoid(-g)
        q, rd, c, _ = swiglu_codes(cfb, gate, up)
        v = g * s * uu
        ok = v.abs() < 3e38                              # beyond: not a finite fp32 number
        a = torch.clamp(v.abs(), min=1e-12)
        # the descale is the one value's magnitude over 448 (or the floor's), the code +-448 (or, far below the floor, zero)
        assert (rd[:, 0].double() * 448 - a)[ok].abs().le((SWIGLU_SLACK + 4 * U) * a[ok] + FLUSHED * abs(u)).all(), u
        got = decode(q, False)[:, 7] * rd[:, 0].double()
        # the code is off by half a step of the coding at the floor: 2^-10 times 1e-12 / 448
        assert (got - v)[ok].abs().le((SWIGLU_SLACK + 8 * U) * v[ok].abs() + FLUSHED * abs(u) + HALF[False] * v[ok].abs() * (v[ok].abs() < 1e-12)
                                      + TINY[False] * 1e-12 / 448).all(), u
        b8, bd = torch.empty((n, 2 * G), dtype=torch.uint8, device="cuda"), torch.empty((n, 2), device="cuda")
        cfb.swiglu_backward_quantize_block128(gate, up, dh, b8, bd)
        got = decode(b8, False)[:, [7, G + 7]] * bd.double()
        # 1 + g (1 - s): the two terms' magnitudes, where they cancel the error is relative to them
        want = torch.stack([d * uu * s * (1 + g * rest), d * g * s], 1)
        size = torch.stack([(d * uu).abs() * s * (1 + (g * rest).abs()), want[:, 1].abs()], 1)
        room = torch.stack([(d * uu).abs(), d.abs()], 1) * FLUSHED
        ok = want.abs() < 3e38
        assert (got - want)[ok].abs().le(((SWIGLU_SLACK + 8 * U) * size + room + HALF[False] * want.abs() * (want.abs() < 1e-12)
                                          + TINY[False] * 1e-12 / 448)[ok]).all(), u


def test_swiglu_gates_without_a_value(cfb):
    """A NaN gate, and an infinite one where the formula has no value (inf * 0): NaN, in forward and gradient, and nowhere else."""
    gate, up, dh = normal((3, 256), 25, 2.0), normal((3, 256), 26), normal((3, 256), 27)
    gate[1, 5], gate[1, 200], gate[2, 9] = float("nan"), float("-inf"), float("inf")
    q, rd, c, cd = swiglu_codes(cfb, gate, up)
    v = decode(q, False)
    assert v[1, 5].isnan() and v[1, 200].isnan() and decode(c, False)[1, [5, 200]].isnan().all() and torch.isfinite(cd[:, 200]).all()
    assert torch.isfinite(rd[1]).all() and int(v[1].isnan().sum()) == 2 and torch.isfinite(v[0]).all() and torch.isfinite(v[2, 128:]).all()
    b8, bd = torch.empty((3, 512), dtype=torch.uint8, device="cuda"), torch.empty((3, 4), device="cuda")
    cfb.swiglu_backward_quantize_block128(gate, up, dh, b8, bd)
    b = decode(b8, False)
    assert b[1, [5, 200, 256 + 5, 256 + 200]].isnan().all() and int(b[1].isnan().sum()) == 4 and torch.isfinite(bd[1]).all()
    assert torch.isfinite(b[0]).all() and b[2, 9].isnan() and int(b[2, :256].isnan().sum()) == 1
    assert torch.isinf(bd[2, 2]) and (b[2, 256:384] * bd[2, 2].double()).isnan().all()          # d up = dh * inf


@pytest.mark.parametrize("e5m2", [False, True])
@pytest.mark.parametrize("rows,cols", [(1, 128), (129, 384), (300, 1024)])
def test_swiglu_gradient_quantise(cfb, rows, cols, e5m2):
    gu, dh = normal((rows, 2 * cols), 31, 2.0), normal((rows, cols), 32, 1e-3)
    gate, up = gu[:, :cols], gu[:, cols:]
    row8 = torch.empty((rows, 2 * cols), dtype=torch.uint8, device="cuda")
    rd = cfb.block128_row_descale(rows, 2 * cols)
    col8 = torch.empty_like(row8)
    cd = torch.empty((cdiv(rows, G), 2 * cols), device="cuda")
    cfb.swiglu_backward_quantize_block128(gate, up, dh, row8, rd, col8, cd, is_e5m2=e5m2)
    g, u, d = gate.double().requires_grad_(), up.double().requires_grad_(), dh.double()
    (g * torch.sigmoid(g) * u).backward(d)               # 64-bit differentiation of the definition
    v = torch.cat([g.grad, u.grad], 1)
    # 1 + gate (1 - sig): where the two terms cancel (gate near -1.28) the error is relative to the terms, each below 1.3
    s = torch.sigmoid(gate.double())
    absolute = torch.cat([(d * u.detach()).abs() * s * (1.0 + (gate.double() * (1 - s)).abs()), u.grad.abs()], 1) * SWIGLU_SLACK
    for codes, scale, dim in ((row8, rd, 1), (col8, cd, 0)):
        a, per = groups64(v, dim)
        _, per_abs = groups64(absolute, dim)
        assert (scale.double() - per / FMAX[e5m2]).abs().le((per_abs + 2 * U * per) / FMAX[e5m2]).all()
        want = v / a * FMAX[e5m2]
        bound = torch.maximum(want.abs() * HALF[e5m2], torch.full_like(want, TINY[e5m2])) * (1 + 2.0 ** -10)
        bound = bound + absolute / a * FMAX[e5m2] + want.abs() * (4 * U + SWIGLU_SLACK)
        assert (decode(codes, e5m2) - want).abs().le(bound).all()


def swiglu_codes(cfb, gate, up):
    """Both groupings of silu(gate) * up: codes and descales of the rows, of the columns."""
    rows, cols = gate.shape
    row8, col8 = (torch.empty((rows, cols), dtype=torch.uint8, device="cuda") for _ in range(2))
    rd, cd = torch.empty((rows, cdiv(cols, G)), device="cuda"), torch.empty((cdiv(rows, G), cols), device="cuda")
    cfb.swiglu_quantize_block128(gate, up, row8, rd, col8, cd)
    return row8, rd, col8, cd


@pytest.mark.parametrize("rows,cols", [(4, 256), (130, 264), (2500, 2304)])       # every tile size of the kernel
def test_swiglu_infinite_gate(cfb, rows, cols):
    """silu(+inf) is +inf: its groups get descale +Inf and contribute NaN, every other group is as it would be without it."""
    gate, up = normal((rows, cols), 23, 2.0), normal((rows, cols), 24)
    q0, d0, c0, cd0 = swiglu_codes(cfb, gate, up)
    only0, od0 = torch.empty_like(q0), torch.empty_like(d0)
    cfb.swiglu_quantize_block128(gate, up, only0, od0)
    assert torch.equal(only0, q0) and torch.equal(od0, d0)
    bad = gate.clone()
    bad[1, 5] = float("inf")
    up[1, 5] = -0.25
    q, d, c, cd = swiglu_codes(cfb, bad, up)
    only, od = torch.empty_like(q), torch.empty_like(d)
    cfb.swiglu_quantize_block128(bad, up, only, od)
    assert torch.equal(only, q) and torch.equal(od, d)
    assert torch.isinf(d[1, 0]) and torch.isinf(cd[0, 5])
    assert (decode(q, False)[1, :G] * d[1, 0].double()).isnan().all()
    assert (decode(c, False)[:min(rows, G), 5] * cd[0, 5].double()).isnan().all()
    d[1, 0], cd[0, 5] = d0[1, 0], cd0[0, 5]              # the two groups that hold it
    q[1, :G], c[:G, 5] = q0[1, :G], c0[:G, 5]
    assert torch.equal(d, d0) and torch.equal(q, q0) and torch.equal(c, c0) and torch.equal(cd, cd0)
    bad[1, 5], up[1, 5] = float("inf"), 0.0              # infinity times zero: NaN, which the amax ignores
    q, d, _, _ = swiglu_codes(cfb, bad, up)
    assert torch.isfinite(d).all() and decode(q, False)[1, 5].isnan() and torch.isfinite(decode(q, False)[1, :5]).all()


# ---------------------------------------------------------------- residual + norm
NORM_SHAPES = [(1, 4096), (3, 1), (5, 100), (2, 129), (65, 512), (33, 1000), (7, 4100), (4, 8193), (3, 16384), (700, 2048)]


def norm64(h, gain, eps):
    h = h.double()
    rms = (h.square().mean(1) + eps).sqrt()
    return h / rms[:, None] * gain.double(), rms


@pytest.mark.parametrize("rows,H", NORM_SHAPES)
@pytest.mark.parametrize("residual", [True, False])
def test_add_rmsnorm_quantise(cfb, rows, H, residual):
    eps = 1e-5
    x, r, gain = normal((rows, H), 41), normal((rows, H), 42, 3.0), normal((H,), 43)
    h = torch.empty_like(x) if residual else None
    rms, normed = torch.empty(rows, device="cuda"), torch.empty_like(x)
    out8 = torch.empty((rows, H), dtype=torch.uint8, device="cuda")
    d = cfb.block128_row_descale(rows, H)
    cfb.add_rmsnorm_quantize_block128(x, r if residual else None, gain, h, rms, normed, out8, d, eps=eps)
    want_h = (x.float() + r.float()).to(torch.bfloat16) if residual else x
    if residual:
        assert torch.equal(h, want_h)                    # one fp32 addition, one rounding
    y, rms64 = norm64(want_h, gain, eps)
    # sum of squares: at most 32 products per thread in a row, 5 + 32 additions behind them; root, division and two products
    slack = (32 + 37 + 4) * U
    assert (rms.double() - rms64).abs().le(slack * rms64).all()
    assert (normed.double() - y).abs().le((2.0 ** -8 + slack) * y.abs() + 1e-38).all()
    check_groups(out8, d, y, 1, False, slack)
    # the codes are the correctly rounded t * 448 / max|t| with t = h * gain, exact ties included (a 19-bit over a 16-bit number:
    # representable or 2^-38 from a border at least, and 64 bits tell those apart)
    t = want_h.double() * gain.double()
    a, _ = groups64(t, 1)
    same = out8 == nearest64(t * 448.0 / a, False)
    # the kernel's quotient carries an error of half a unit of fp32: a border closer than 2^-23 may be on the other side
    off = (t * 448.0 / a)[~same]
    near = torch.minimum((nearest64(off * (1 + 2.0 ** -22), False) != nearest64(off * (1 - 2.0 ** -22), False)).double(), torch.ones_like(off))
    assert near.bool().all(), int((~same).sum())
    # in place: h may be the residual, or x; the codes alone and the bf16 row alone are the same
    for into in ("r", "x"):
        xx, rr = x.clone(), r.clone()
        o2, d2 = torch.empty_like(out8), torch.empty((rows, cdiv(H, G)), device="cuda")
        if residual:
            cfb.add_rmsnorm_quantize_block128(xx, rr, gain, rr if into == "r" else xx, None, None, o2, d2, eps=eps)
            assert torch.equal(rr if into == "r" else xx, want_h)
        else:
            cfb.add_rmsnorm_quantize_block128(xx, None, gain, None, None, None, o2, d2, eps=eps)
        assert torch.equal(o2, out8) and torch.equal(d2, d)
    n2 = torch.empty_like(x)
    cfb.add_rmsnorm_quantize_block128(want_h, None, gain, None, None, n2, eps=eps)
    assert torch.equal(n2, normed)


def test_add_rmsnorm_zero_rows_and_row_of_zeros(cfb):
    gain = normal((256,), 1)
    x = torch.zeros((2, 256), dtype=torch.bfloat16, device="cuda")
    out8, d = torch.full((2, 256), 7, dtype=torch.uint8, device="cuda"), torch.empty((2, 2), device="cuda")
    cfb.add_rmsnorm_quantize_block128(x, None, gain, None, None, None, out8, d)
    assert (decode(out8, False) == 0).all() and torch.equal(d, (torch.full_like(d, 1e-12).double() / 448.0).float())
    cfb.add_rmsnorm_quantize_block128(x[:0], None, gain, None, None, None, out8[:0], d[:0])


# one vector per thread, two, four, and rows that are not made of whole vectors
WIDTHS = [(6, 512), (200, 4096), (700, 4096), (5, 16384), (5, 1001)]


@pytest.mark.parametrize("rows,H", WIDTHS)
@pytest.mark.parametrize("residual", [True, False])
def test_add_rmsnorm_infinities_and_nan(cfb, rows, H, residual):
    """A row with an infinity: rms is infinite, its y is 0, NaN at the infinity itself; a row with a NaN: NaN throughout. Groups
    without a finite value other than zero get the descale of the floor. The rows beside them are as they would be alone."""
    x, r, gain = normal((rows, H), 45), normal((rows, H), 46), normal((H,), 47)

    def run(x):
        h, normed, rms = (torch.empty_like(x) if residual else None), torch.empty_like(x), torch.empty(rows, device="cuda")
        out8, d = torch.empty((rows, H), dtype=torch.uint8, device="cuda"), torch.empty((rows, cdiv(H, G)), device="cuda")
        cfb.add_rmsnorm_quantize_block128(x, r if residual else None, gain, h, rms, normed, out8, d)
        return (x if h is None else h), normed, rms, decode(out8, False), d
    h0, n0, rms0, v0, d0 = run(x)
    bad = x.clone()
    bad[1, 3], bad[2, H - 1], bad[3, 130] = float("inf"), float("-inf"), float("nan")
    h, n, rms, v, d = run(bad)
    assert torch.isinf(h[1, 3]) and torch.isinf(h[2, H - 1]) and h[3, 130].isnan()
    assert torch.isinf(rms[1:3]).all() and rms[3].isnan()
    floor = float((torch.tensor(1e-12).double() / 448.0).float())
    for row, at in ((1, 3), (2, H - 1)):
        rest = torch.arange(H, device="cuda") != at
        assert v[row, at].isnan() and v[row][rest].eq(0).all() and d[row].eq(floor).all()
        assert n[row, at].isnan() and n[row][rest].eq(0).all()
    assert v[3].isnan().all() and n[3].isnan().all() and d[3].eq(floor).all()
    rest = torch.ones(rows, dtype=torch.bool, device="cuda")
    rest[1:4] = False
    for a, b in ((n, n0), (rms, rms0), (v, v0), (d, d0)):
        assert torch.equal(a[rest], b[rest])


@pytest.mark.parametrize("rows,H", WIDTHS)
@pytest.mark.parametrize("residual", [True, False])
def test_add_rmsnorm_rows_whose_squares_overflow(cfb, rows, H, residual):
    """Finite values above 1.8e19 have squares beyond fp32: rms, y and codes are right all the same."""
    eps = 1e-6
    x, gain = normal((rows, H), 48), normal((H,), 49)
    r = normal((rows, H), 44)
    x[0] *= 1e30                                         # all of the row
    x[1, 3] = 2e19                                       # one value, the others vanish beside it
    x[2] = 3.3895e38                                     # the largest bf16 number throughout
    x[3, H - 1], x[3, 0] = -3.3895e38, 1e25
    x[4, : H // 2] *= 1e18                               # the sum overflows, no square does
    r[2] = 0.0
    rms, normed, h = torch.empty(rows, device="cuda"), torch.empty_like(x), torch.empty_like(x) if residual else None
    out8, d = torch.empty((rows, H), dtype=torch.uint8, device="cuda"), torch.empty((rows, cdiv(H, G)), device="cuda")
    cfb.add_rmsnorm_quantize_block128(x, r if residual else None, gain, h, rms, normed, out8, d, eps=eps)
    want_h = (x.float() + r.float()).to(torch.bfloat16) if residual else x
    assert h is None or torch.equal(h, want_h)
    y, rms64 = norm64(want_h, gain, eps)
    # as for ordinary rows: 32 squares per thread, 37 additions behind them, root, quotient and products
    slack = (32 + 37 + 4) * U
    assert torch.isfinite(rms).all() and (rms.double() - rms64).abs().le(slack * rms64).all()
    assert (normed.double() - y).abs().le((2.0 ** -8 + slack) * y.abs() + 1e-38).all()
    check_groups(out8, d, y, 1, False, slack)
    only, od = torch.empty_like(out8), torch.empty_like(d)           # in place, the codes alone
    cfb.add_rmsnorm_quantize_block128(x, r if residual else None, gain, x if residual else None, None, None, only, od, eps=eps)
    assert torch.equal(only, out8) and torch.equal(od, d)


def grad64(dy, h, gain, rms, dh):
    dy, xh, g = dy.double(), h.double() / rms.double()[:, None], gain.double()
    u = dy * g
    dx = (u - xh * (u * xh).mean(1, keepdim=True)) / rms.double()[:, None]
    return dx + (0 if dh is None else dh.double()), (dy * xh).sum(0)


@pytest.mark.parametrize("rows,H", NORM_SHAPES + [(1500, 256)])
@pytest.mark.parametrize("with_dh", [True, False])
def test_add_rmsnorm_gradient(cfb, rows, H, with_dh):
    eps = 1e-5
    h, gain, dy = normal((rows, H), 51, 2.0), normal((H,), 52), normal((rows, H), 53, 1e-2)
    dh = normal((rows, H), 54, 1e-2) if with_dh else None
    rms = (h.double().square().mean(1) + eps).sqrt().float()
    dx, dg = torch.empty_like(h), torch.full((H,), 3.0, device="cuda")
    scratch = torch.full((cfb.add_rmsnorm_backward_scratch_floats(rows, H),), float("nan"), device="cuda")
    cfb.add_rmsnorm_backward(dy, h, gain, rms, dh, dx, dg, scratch)
    want_dx, want_dg = grad64(dy, h, gain, rms, dh)
    # dx: bf16 rounding of the result; the mean is a sum of H products with the error of its absolute terms
    xh = (h.double() / rms.double()[:, None]).abs()
    u = (dy.double() * gain.double()).abs()
    terms = (u + xh * (u * xh).mean(1, keepdim=True)) / rms.double()[:, None] + (0 if dh is None else dh.double().abs())
    assert (dx.double() - want_dx).abs().le(2.0 ** -8 * want_dx.abs() + (32 + 37 + 8) * U * terms + 1e-38).all()
    # dgain: per block at most rows / blocks products in a row, then at most 592 / 32 + 32 partial sums
    depth = cdiv(rows, 148) + 19 + 32 + 4
    assert (dg.double() - want_dg).abs().le(depth * U * (dy.double() * h.double() / rms.double()[:, None]).abs().sum(0)).all()
    # accumulated on top; the same bits on every call; in place of either gradient; without the gain's gradient
    dg2 = dg.clone()
    into = dy.clone()
    cfb.add_rmsnorm_backward(into, h, gain, rms, dh, into, dg2, scratch, accumulate_dscale=True)
    assert torch.equal(into, dx) and torch.equal(dg2, dg + dg)
    if with_dh:
        into = dh.clone()
        cfb.add_rmsnorm_backward(dy, h, gain, rms, into, into)
        assert torch.equal(into, dx)


# every number of vectors a thread holds (by row length and by row count), and blocks that walk several rows
@pytest.mark.parametrize("rows,H", [(148, 520), (149, 4096), (593, 4096), (15000, 128), (1800, 4104), (1800, 8192), (460, 8200), (300, 4101)])
def test_add_rmsnorm_many_rows(cfb, rows, H):
    test_add_rmsnorm_quantise(cfb, rows, H, True)
    test_add_rmsnorm_gradient(cfb, rows, H, True)


def test_add_rmsnorm_gradient_against_differences(cfb):
    """A directional derivative of sum(c * y(h)) in 64 bits against the kernel's gradient."""
    rows, H, eps = 4, 512, 1e-5
    h, gain, c, t = normal((rows, H), 61), normal((H,), 62), normal((rows, H), 63), normal((rows, H), 64).double()
    tg = normal((H,), 65).double()
    rms = norm64(h, gain, eps)[1].float()
    dx, dg = torch.empty_like(h), torch.empty(H, device="cuda")
    scratch = torch.empty(cfb.add_rmsnorm_backward_scratch_floats(rows, H), device="cuda")
    cfb.add_rmsnorm_backward(c, h, gain, rms, None, dx, dg, scratch)

    def f(e, eg):
        hh, g = h.double() + e * t, gain.double() + eg * tg
        return (c.double() * hh / (hh.square().mean(1, keepdim=True) + eps).sqrt() * g).sum()
    s = 1e-5
    dh_num, dg_num = (f(s, 0) - f(-s, 0)) / (2 * s), (f(0, s) - f(0, -s)) / (2 * s)
    # dx is rounded to bf16: 2^-8 of every term; the difference quotient is good to s^2 and 1e-16 / s of the sum
    tol = 2.0 ** -8 * (dx.double() * t).abs().sum() + 1e-6 * (c.double() * t).abs().sum()
    assert (dh_num - (dx.double() * t).sum()).abs() <= tol
    assert (dg_num - (dg.double() * tg).sum()).abs() <= 1e-5 * (dg.double() * tg).abs().sum()


# ---------------------------------------------------------------- products
def coded(rows, cols, seed, rows_per, cols_per, e5m2=False, std=1.0):
    """Random codes (finite, over the whole range of the type) with a pitch that is a multiple of 16, and random descales."""
    v = (torch.randn((rows, cols), generator=gen(seed), device="cuda") * std * 60).clamp(-FMAX[e5m2], FMAX[e5m2])
    buf = torch.full((rows, cdiv(cols, 16) * 16), 0x7f, dtype=torch.uint8, device="cuda")     # NaN behind the columns: not to be read
    buf[:, :cols] = v.to(TYPE[e5m2]).view(torch.uint8)
    d = torch.rand((cdiv(rows, rows_per), cdiv(cols, cols_per)), generator=gen(seed + 1), device="cuda") * 0.02 + 1e-4
    return buf[:, :cols], d


def value64(codes, d, e5m2, rows_per, cols_per):
    R, C = codes.shape
    d = d.double().repeat_interleave(rows_per, 0)[:R].repeat_interleave(cols_per, 1)[:, :C]
    return decode(codes, e5m2) * d


def check_product(out, a, b, K, before=None):
    """out = a . b (64 bits) up to fp32 sums and one rounding to out's type."""
    want, mag = a @ b, a.abs() @ b.abs()
    if before is not None:
        want, mag = want + before, mag + before.abs()
    # a block's 128 products are exact and added in fp32 (one unit of 2^-23 each at most); then per block the two scales'
    # product, its product with the block and one addition
    fp32 = (128 * 2 + 3 * cdiv(K, G) + 2) * U
    half = 2.0 ** -8 if out.dtype == torch.bfloat16 else U
    err = (out.double() - want).abs()
    assert torch.isfinite(out).all()
    bound = half * want.abs() + fp32 * mag
    assert err.le(bound).all(), float((err / bound.clamp(min=1e-300)).max())


NT_SHAPES = [(1, 1, 1), (1, 4096, 4096), (2, 100, 200), (16, 256, 128), (17, 129, 384), (33, 520, 1000), (64, 384, 2048),
             (100, 128, 144), (128, 1000, 640), (129, 256, 128), (200, 64, 100), (300, 520, 1000), (513, 260, 272),
             (777, 1000, 520), (512, 512, 4096), (1100, 2304, 1024)]


@pytest.mark.parametrize("M,N,K", NT_SHAPES)
def test_product_nt(cfb, ctx, M, N, K):
    A, da = coded(M, K, M + N, 1, G)
    B, db = coded(N, K, M + K, G, G, std=0.5)
    out = torch.empty((M, N), dtype=torch.bfloat16, device="cuda")
    cfb.gemm_fp8_block128_nt(ctx, A, da, B, db, out)
    ctx.poll_status()
    a, b = value64(A, da, False, 1, G), value64(B, db, False, G, G).t()
    check_product(out, a, b, K)
    # fp32 output, stored and added to; descales with the rows next to each other; the same sums
    f = torch.full((M, N), 5.0, device="cuda")
    cfb.gemm_fp8_block128_nt(ctx, A, da.t().contiguous().t(), B, db, f)
    check_product(f, a, b, K)
    assert torch.equal(f.to(torch.bfloat16), out)
    g = f.clone()
    cfb.gemm_fp8_block128_nt(ctx, A, da, B, db, g, accumulate=True)
    assert torch.equal(g, f + f)
    c = normal((M, N), 9, 10.0)
    c0 = c.clone()
    cfb.gemm_fp8_block128_nt(ctx, A, da, B, db, c, accumulate=True)
    assert torch.equal(c, (c0.float() + f).to(torch.bfloat16))
    ctx.poll_status()


@pytest.mark.parametrize("M,N,K", [(5, 300, 520), (130, 260, 272), (600, 300, 400)])
def test_product_nt_types_row_groups_and_pitches(cfb, ctx, M, N, K):
    A, da = coded(M, K, 1, 1, G, e5m2=True)
    B, db = coded(N, K, 2, 1, G)
    a, b = value64(A, da, True, 1, G), value64(B, db, False, 1, G).t()
    for pad, offset in ((0, 0), (1, 0), (8, 8), (3, 1)):
        out, raw = pitched(M, N, torch.bfloat16, pad, offset)
        cfb.gemm_fp8_block128_nt(ctx, A, da, B, db, out, a_is_e5m2=True)
        check_product(out, a, b, K)
        out.copy_(torch.full((), 0x5a5a, dtype=torch.int16, device="cuda").view(torch.bfloat16))
        assert raw.eq(0x5a).all()                        # nothing between or behind the rows was written
        f, raw = pitched(M, N, torch.float32, pad, offset)
        cfb.gemm_fp8_block128_nt(ctx, A, da, B, db, f, a_is_e5m2=True)
        check_product(f, a, b, K)
        f.copy_(torch.full((), 0x5a5a5a5a, dtype=torch.int32, device="cuda").view(torch.float32))
        assert raw.eq(0x5a).all()
    ctx.poll_status()


def test_product_scale_extremes(cfb, ctx):
    """Scales far apart between blocks, zero scales, and a NaN or infinite scale that reaches its own row or column only."""
    for M in (8, 300):
        N, K = 384, 512
        A, da = coded(M, K, 3, 1, G)
        B, db = coded(N, K, 4, G, G)
        da[:, 1] *= 1e6
        da[:, 2] = 0.0
        db[1, 3] = 0.0
        out = torch.empty((M, N), device="cuda")
        cfb.gemm_fp8_block128_nt(ctx, A, da, B, db, out)
        check_product(out, value64(A, da, False, 1, G), value64(B, db, False, G, G).t(), K)
        da[5, 0], db[2, 3] = float("nan"), float("inf")
        cfb.gemm_fp8_block128_nt(ctx, A, da, B, db, out)
        assert out[5].isnan().all() and not torch.isfinite(out[:, 256:]).any()
        rest = torch.ones(M, dtype=torch.bool, device="cuda")
        rest[5] = False
        check_product(out[rest][:, :256], value64(A, da, False, 1, G)[rest], value64(B, db, False, G, G)[:256].t(), K)


@pytest.mark.parametrize("counts,gap,tail", [([5, 0, 130, 1], 0, 3), ([300, 257, 0, 0, 40], 2, 0), ([0, 0], 0, 4), ([1], 0, 0),
                                             ([700, 600, 513], 1, 9), ([3] * 130, 0, 1)])
@pytest.mark.parametrize("N,K", [(256, 256), (200, 520)])
def test_product_grouped(cfb, ctx, counts, gap, tail, N, K):
    E = len(counts)
    offsets = np.cumsum([0] + [c + gap for c in counts[:-1]])
    T = int(offsets[-1]) + counts[-1] + tail
    A, da = coded(T, K, 5, 1, G)
    stack = [coded(N, K, 100 + 2 * e, G, G) for e in range(E)]
    B = torch.stack([torch.nn.functional.pad(s[0], (0, -K % 16)) for s in stack])[..., :K]
    db = torch.stack([s[1] for s in stack])
    ct = torch.tensor(counts, dtype=torch.int32, device="cuda")
    ot = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    out, raw = pitched(T, N, torch.bfloat16, 8)
    cfb.gemm_fp8_block128_nt_grouped(ctx, ct, ot, A, da, B, db, out)
    ctx.poll_status()
    a = value64(A, da, False, 1, G)
    for e, (o, n) in enumerate(zip(offsets, counts)):
        if n:
            check_product(out[o:o + n], a[o:o + n], value64(B[e], db[e], False, G, G).t(), K)
            out[o:o + n] = torch.full((), 0x5a5a, dtype=torch.int16, device="cuda").view(torch.bfloat16)
    assert raw.eq(0x5a).all()                            # rows of no group, and everything between the rows, as they were


def test_product_grouped_counts_that_leave_the_buffer(cfb, ctx):
    """Device counts and offsets are not trusted: a group is cut to the buffer, one that starts outside is skipped."""
    T, N, K, E = 140, 256, 256, 4
    A, da = coded(T, K, 5, 1, G)
    stack = [coded(N, K, 200 + 2 * e, G, G) for e in range(E)]
    B, db = torch.stack([s[0] for s in stack]), torch.stack([s[1] for s in stack])
    out, raw = pitched(T, N, torch.bfloat16, 0)
    cfb.gemm_fp8_block128_nt_grouped(ctx, torch.tensor([10, 1000, 5, -7], dtype=torch.int32, device="cuda"),
                                     torch.tensor([0, 20, 5000, 12], dtype=torch.int32, device="cuda"), A, da, B, db, out)
    ctx.poll_status()
    a = value64(A, da, False, 1, G)
    check_product(out[:10], a[:10], value64(B[0], db[0], False, G, G).t(), K)
    check_product(out[20:], a[20:], value64(B[1], db[1], False, G, G).t(), K)
    assert raw.view(torch.bfloat16)[10 * N:20 * N].view(torch.int16).eq(0x5a5a).all()
    assert raw[T * N * 2:].eq(0x5a).all()


@pytest.mark.parametrize("e5m2", [False, True])
@pytest.mark.parametrize("M,N,K", [(1, 16, 1), (100, 200, 130), (300, 128, 520), (513, 1000, 256), (700, 272, 1100), (512, 512, 4096)])
def test_product_nn(cfb, ctx, M, N, K, e5m2):
    A, da = coded(M, K, 6, 1, G, e5m2=e5m2)
    B, db = coded(K, N, 7, G, G)
    out = torch.empty((M, N), dtype=torch.bfloat16, device="cuda")
    cfb.gemm_fp8_block128_nn(ctx, A, da, B, db, out, a_is_e5m2=e5m2)
    ctx.poll_status()
    a, b = value64(A, da, e5m2, 1, G), value64(B, db, False, G, G)
    check_product(out, a, b, K)
    f = torch.zeros((M, N), device="cuda")
    cfb.gemm_fp8_block128_nn(ctx, A, da, B, db, f, a_is_e5m2=e5m2, accumulate=True)
    assert torch.equal(f.to(torch.bfloat16), out)


@pytest.mark.parametrize("xe,ye", [(False, True), (False, False), (True, False)])
@pytest.mark.parametrize("M,N,T", [(16, 16, 1), (256, 300, 100), (100, 520, 130), (513, 260, 640), (1000, 272, 1100), (512, 768, 4096)])
def test_product_dw(cfb, ctx, M, N, T, xe, ye):
    X, dx = coded(T, M, 8, G, 1, e5m2=xe)
    Y, dy = coded(T, N, 9, G, 1, e5m2=ye)
    f = torch.full((M, N), 2.0, device="cuda")
    cfb.gemm_fp8_block128_dw(ctx, X, dx, Y, dy, f, x_is_e5m2=xe, dy_is_e5m2=ye)
    ctx.poll_status()
    x, y = value64(X, dx, xe, G, 1).t(), value64(Y, dy, ye, G, 1)
    check_product(f, x, y, T)
    g = f.clone()
    cfb.gemm_fp8_block128_dw(ctx, X, dx, Y, dy, g, x_is_e5m2=xe, dy_is_e5m2=ye, accumulate=True)
    assert torch.equal(g, f + f)
    h = torch.empty((M, N), dtype=torch.bfloat16, device="cuda")
    cfb.gemm_fp8_block128_dw(ctx, X, dx.t().contiguous().t(), Y, dy.t().contiguous().t(), h, x_is_e5m2=xe, dy_is_e5m2=ye)
    assert torch.equal(h, f.to(torch.bfloat16))
    c = normal((M, N), 10)
    c0 = c.clone()
    cfb.gemm_fp8_block128_dw(ctx, X, dx, Y, dy, c, x_is_e5m2=xe, dy_is_e5m2=ye, accumulate=True)
    assert torch.equal(c, (c0.float() + f).to(torch.bfloat16))


# More tiles than the chip holds at once, so that every CTA goes from tile to tile (the stages, barrier phases, TMEM buffers and
# output boxes carry over): CTA pairs with five tiles each, single CTAs with two; an even and an odd number of blocks of K, and one
SEVERAL_TILES = [(4999, 4360, 100), (4999, 4360, 400), (4999, 4360, 528), (300, 20000, 300), (300, 20000, 128)]


@pytest.mark.parametrize("row_groups", [False, True])
@pytest.mark.parametrize("M,N,K", SEVERAL_TILES)
def test_product_nt_several_tiles_each(cfb, ctx, M, N, K, row_groups):
    per = 1 if row_groups else G
    A, da = coded(M, K, M + N, 1, G)
    B, db = coded(N, K, M + K, per, G, std=0.5)
    a, b = value64(A, da, False, 1, G), value64(B, db, False, per, G).t()
    out, f = torch.empty((M, N), dtype=torch.bfloat16, device="cuda"), torch.full((M, N), 5.0, device="cuda")
    cfb.gemm_fp8_block128_nt(ctx, A, da, B, db, out)
    cfb.gemm_fp8_block128_nt(ctx, A, da.t().contiguous().t(), B, db, f)
    ctx.poll_status()
    check_product(f, a, b, K)
    assert torch.equal(out, f.to(torch.bfloat16))
    del a, b
    for pad in (0, 1):                                   # whole boxes, and element by element
        for dtype in (torch.float32, torch.bfloat16):
            o, raw = pitched(M, N, dtype, pad)
            cfb.gemm_fp8_block128_nt(ctx, A, da, B, db, o)
            assert torch.equal(o, f.to(dtype))
            cfb.gemm_fp8_block128_nt(ctx, A, da, B, db, o, accumulate=True)
            assert torch.equal(o, (f.to(dtype).float() + f).to(dtype))
            o.copy_(torch.full((), 0x5a5a if dtype == torch.bfloat16 else 0x5a5a5a5a, device="cuda",
                               dtype=torch.int16 if dtype == torch.bfloat16 else torch.int32).view(dtype))
            assert raw.eq(0x5a).all()
    ctx.poll_status()


@pytest.mark.parametrize("counts,tail", [([2431, 2600], 89), ([300, 0, 129, 1, 128, 257, 400, 90, 183], 12)])
@pytest.mark.parametrize("K", [300, 400])
def test_product_grouped_several_tiles_each(cfb, ctx, counts, tail, K):
    """CTA pairs (two large groups) and single CTAs (nine small ones)."""
    N, E = 4352, len(counts)
    offsets = np.cumsum([0] + counts[:-1])
    T = sum(counts) + tail
    A, da = coded(T, K, 5, 1, G)
    stack = [coded(N, K, 300 + 2 * e, G, G) for e in range(E)]
    B = torch.stack([torch.nn.functional.pad(s[0], (0, -K % 16)) for s in stack])[..., :K]
    db = torch.stack([s[1] for s in stack])
    ct, ot = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in (counts, offsets))
    a = value64(A, da, False, 1, G)
    for pad in (0, 8, 3):
        out, raw = pitched(T, N, torch.bfloat16, pad)
        cfb.gemm_fp8_block128_nt_grouped(ctx, ct, ot, A, da, B, db, out)
        ctx.poll_status()
        for e, (o, n) in enumerate(zip(offsets, counts)):
            if n:
                check_product(out[o:o + n], a[o:o + n], value64(B[e], db[e], False, G, G).t(), K)
                out[o:o + n] = torch.full((), 0x5a5a, dtype=torch.int16, device="cuda").view(torch.bfloat16)
        assert raw.eq(0x5a).all()


def test_product_gradients_several_tiles_each(cfb, ctx):
    """Data and weight gradient with two or three tiles to a CTA pair and an odd number of blocks."""
    M, N, K = 2300, 4112, 300
    A, da = coded(M, K, 16, 1, G, e5m2=True)
    B, db = coded(K, N, 17, G, G)
    for pad in (0, 1):
        f, _ = pitched(M, N, torch.float32, pad)
        cfb.gemm_fp8_block128_nn(ctx, A, da, B, db, f, a_is_e5m2=True)
        check_product(f, value64(A, da, True, 1, G), value64(B, db, False, G, G), K)
        out, _ = pitched(M, N, torch.bfloat16, pad)
        cfb.gemm_fp8_block128_nn(ctx, A, da, B, db, out, a_is_e5m2=True)
        assert torch.equal(out, f.to(torch.bfloat16))
    M, T = 2304, 620
    X, dx = coded(T, M, 18, G, 1)
    Y, dy = coded(T, N, 19, G, 1, e5m2=True)
    for pad in (0, 1):
        f, _ = pitched(M, N, torch.float32, pad)
        cfb.gemm_fp8_block128_dw(ctx, X, dx, Y, dy, f, dy_is_e5m2=True)
        check_product(f, value64(X, dx, False, G, 1).t(), value64(Y, dy, True, G, 1), T)
        g = f.clone()
        cfb.gemm_fp8_block128_dw(ctx, X, dx, Y, dy, g, dy_is_e5m2=True, accumulate=True)
        assert torch.equal(g, f + f)
    ctx.poll_status()


@pytest.mark.parametrize("M,N,K", [(8500, 17000, 4096), (4200, 16000, 4224)])
def test_product_nt_weights_larger_than_the_cache(cfb, ctx, M, N, K):
    """Products that walk their tiles in bands of 32 and of 16 row blocks, one band and a piece: rows of every block against 64 bits."""
    A, da = coded(M, K, M + N, 1, G)
    B, db = coded(N, K, M + K, G, G, std=0.5)
    out = torch.empty((M, N), dtype=torch.bfloat16, device="cuda")
    cfb.gemm_fp8_block128_nt(ctx, A, da, B, db, out)
    ctx.poll_status()
    rows = torch.cat([torch.arange(3, M, 128, device="cuda"), torch.tensor([0, M - 1], device="cuda")])     # both CTAs of every pair
    check_product(out[rows], value64(A[rows], da[rows], False, 1, G), value64(B, db, False, G, G).t(), K)


def test_empty_sizes_do_nothing(cfb, ctx):
    A, da = coded(4, 256, 1, 1, G)
    B, db = coded(128, 256, 2, G, G)
    cfb.gemm_fp8_block128_nt(ctx, A[:0], da[:0], B, db, torch.empty((0, 128), dtype=torch.bfloat16, device="cuda"))
    x = normal((0, 256), 1)
    cfb.fp8_quantize_block128(x, torch.empty((0, 256), dtype=torch.uint8, device="cuda"), torch.empty((0, 2), device="cuda"))
    dg = torch.ones(256, device="cuda")
    cfb.add_rmsnorm_backward(x, x, normal((256,), 1), torch.empty(0, device="cuda"), None, x, dg, torch.empty(0, device="cuda"))
    assert dg.eq(0).all()
    cfb.add_rmsnorm_backward(x, x, normal((256,), 1), torch.empty(0, device="cuda"), None, x, dg.fill_(1), torch.empty(0, device="cuda"),
                             accumulate_dscale=True)
    assert dg.eq(1).all()


def test_empty_contraction_is_zero(cfb, ctx):
    for dtype in (torch.bfloat16, torch.float32):
        out, raw = pitched(5, 100, dtype, 3)
        out.fill_(2.0)
        kept = raw.clone()
        A, da, B, db = (torch.empty(s, dtype=t, device="cuda") for s, t in (((5, 0), torch.uint8), ((5, 0), torch.float32), ((100, 0), torch.uint8), ((1, 0), torch.float32)))
        cfb.gemm_fp8_block128_nt(ctx, A, da, B, db, out, accumulate=True)
        assert torch.equal(raw, kept)
        cfb.gemm_fp8_block128_nt(ctx, A, da, B, db, out)
        assert out.eq(0).all()
        out.fill_(2.0)
        X, dx, Y, dy = (torch.empty(s, dtype=t, device="cuda") for s, t in (((0, 5), torch.uint8), ((0, 5), torch.float32), ((0, 100), torch.uint8), ((0, 100), torch.float32)))
        cfb.gemm_fp8_block128_dw(ctx, X, dx, Y, dy, out)
        assert out.eq(0).all()
        out.fill_(2.0)
        assert torch.equal(raw, kept)                    # nothing beside the matrix was written


@pytest.mark.parametrize("pad,offset", [(1, 0), (8, 8), (3, 5)])
def test_swiglu_pitches_and_alignments(cfb, pad, offset):
    rows, cols = 141, 256
    (gate, _), (up, _), (dh, _) = (pitched(rows, cols, torch.bfloat16, pad, offset) for _ in range(3))
    for i, t in enumerate((gate, up, dh)):
        t.copy_(normal((rows, cols), 140 + i))
    even = [t.contiguous() for t in (gate, up, dh)]

    def run(g, u, d, view):
        q, qc = view(cols), view(cols)
        rd, cd = torch.empty((rows, 2), device="cuda"), torch.empty((2, cols), device="cuda")
        cfb.swiglu_quantize_block128(g, u, q, rd, qc, cd)
        b, bc = view(2 * cols), view(2 * cols)
        bd, bcd = torch.empty((rows, 4), device="cuda"), torch.empty((2, 2 * cols), device="cuda")
        cfb.swiglu_backward_quantize_block128(g, u, d, b, bd, bc, bcd)
        alone, ad = view(2 * cols), torch.empty((rows, 4), device="cuda")
        cfb.swiglu_backward_quantize_block128(g, u, d, alone, ad)
        calone, cad = view(2 * cols), torch.empty((2, 2 * cols), device="cuda")
        cfb.swiglu_backward_quantize_block128(g, u, d, col8=calone, col_descale=cad)
        assert torch.equal(alone, b) and torch.equal(ad, bd) and torch.equal(calone, bc) and torch.equal(cad, bcd)
        return q, rd, qc, cd, b, bd, bc, bcd

    odd = run(gate, up, dh, lambda c: pitched(rows, c, torch.uint8, pad, offset)[0])
    plain = run(*even, lambda c: torch.empty((rows, c), dtype=torch.uint8, device="cuda"))
    assert all(torch.equal(a, b) for a, b in zip(odd, plain))


def test_offsets_beyond_32_bits(cfb, ctx):
    """Rows whose elements lie more than 2^32 apart from the first one: quantisers, both forms of the product, all outputs."""
    free, _ = torch.cuda.mem_get_info()
    if free < 60 << 30:
        pytest.skip("needs 60 GB of device memory")
    rows, cols, far = 4, 256, 1_600_000_000              # 3 * far elements > 2^32
    big = torch.empty(rows * far, dtype=torch.uint8, device="cuda")
    q = big.view(rows, far)[:, :cols]
    x = normal((rows, cols), 150)
    rd, cd = torch.empty((rows, 2), device="cuda"), torch.empty((1, cols), device="cuda")
    cfb.fp8_quantize_block128(x, q, rd)
    want, _ = plain_codes(x, 1, False)
    assert torch.equal(q, want)
    B, db = coded(384, cols, 151, G, G)
    out = torch.empty((rows, 384), device="cuda")
    cfb.gemm_fp8_block128_nt(ctx, q, rd, B, db, out)     # narrow form, A far apart
    check_product(out, value64(q, rd, False, 1, G), value64(B, db, False, G, G).t(), cols)
    cfb.fp8_quantize_block128(x, col8=q, col_descale=cd)
    want, _ = plain_codes(x, 0, False)
    assert torch.equal(q, want)
    del big, q
    M, N, far = 300, 384, 16_000_000                     # 299 * far elements > 2^32
    big = torch.empty(M * far, dtype=torch.bfloat16, device="cuda")
    out = big.view(M, far)[:, :N]
    A, da = coded(M, cols, 152, 1, G)
    for n in (M, 40):                                    # wide and narrow form, output rows far apart
        cfb.gemm_fp8_block128_nt(ctx, A[:n], da[:n], B, db, out[:n] if n == M else out[M - n:])
        check_product(out[:n] if n == M else out[M - n:], value64(A[:n], da[:n], False, 1, G), value64(B, db, False, G, G).t(), cols)
    xin = out[:, :cols]
    xin.copy_(normal((M, cols), 153))
    q = torch.empty((M, cols), dtype=torch.uint8, device="cuda")
    rd = torch.empty((M, 2), device="cuda")
    cfb.fp8_quantize_block128(xin, q, rd)                # input rows far apart
    want, d = plain_codes(xin, 1, False)
    assert torch.equal(q, want) and torch.equal(rd, d)
    ctx.poll_status()


# ---------------------------------------------------------------- run together
def rel(a, b):
    a, b = a.detach().double(), b.detach().double()
    return float((a - b).norm() / b.norm())


@pytest.mark.parametrize("rows,H,F", [(1, 256, 384), (37, 512, 256), (300, 256, 640), (1000, 512, 1024)])
def test_feed_forward_block_forward_and_gradients(cfb, ctx, rows, H, F):
    """The block's stages against 64 bits on the codes that each of them really read, and the whole against 64-bit
    differentiation of the block without any coding."""
    x, r = normal((rows, H), 71), normal((rows, H), 72)
    gain = (1 + 0.1 * torch.randn(H, generator=gen(73), device="cuda")).to(torch.bfloat16)
    wgu, wd = cfb.Fp8Block128Weight(normal((2 * F, H), 74, H ** -0.5)), cfb.Fp8Block128Weight(normal((H, F), 75, F ** -0.5))
    dy, dh = normal((rows, H), 76, 1e-2), normal((rows, H), 77, 1e-2)
    block = cfb.FfnSwigluFp8Block128(ctx, rows + 5, H, F, train=True)
    y, dx = torch.empty_like(x), torch.empty_like(x)
    dwgu, dwd, dg = torch.empty((2 * F, H), device="cuda"), torch.empty((H, F), device="cuda"), torch.empty(H, device="cuda")
    block.forward(x, r, gain, wgu, wd, y)
    block.backward(dy, dh, gain, wgu, wd, dx, dwgu, dwd, dg)
    ctx.poll_status()
    n8, dn8 = block._rows(block.n8)
    Wgu, Wd = value64(wgu.w8, wgu.descale, False, G, G), value64(wd.w8, wd.descale, False, G, G)
    check_product(block.gu[:rows], value64(n8, dn8, False, 1, G), Wgu.t(), H)
    check_product(y, value64(*block._rows(block.a8), False, 1, G), Wd.t(), F)
    check_product(block.da[:rows], value64(*block._rows(block.dy8), True, 1, G), Wd, H)
    check_product(dwd, value64(*block._cols(block.dy8c), True, G, 1).t(), value64(*block._cols(block.a8c), False, G, 1), rows)
    check_product(block.dn[:rows], value64(*block._rows(block.dgu8), True, 1, G), Wgu, 2 * F)
    check_product(dwgu, value64(*block._cols(block.dgu8c), True, G, 1).t(), value64(*block._cols(block.n8c), False, G, 1), rows)
    # without coding: X, W and the gradients in 64 bits
    leaves = [t.double().requires_grad_() for t in (x, gain, wgu.w, wd.w)]
    X, gg, Wg, Wo = leaves
    h = X + r.double()
    n = h / (h.square().mean(1, keepdim=True) + 1e-6).sqrt() * gg
    gu = n @ Wg.t()
    out = (torch.nn.functional.silu(gu[:, :F]) * gu[:, F:]) @ Wo.t()
    (out * dy.double()).sum().backward(retain_graph=True)
    h.backward(dh.double())
    # a code is off by 2^-4 of its value at most and 2.6 % rms (E4M3; 5.2 % for E5M2), independently from element to element;
    # the longest way passes four E4M3 and two E5M2 codings: sqrt(4 * 2.6^2 + 2 * 5.2^2) = 9 %, two of these are allowed
    for got, want, limit in ((y, out, 0.105), (dx, X.grad, 0.18), (dg, gg.grad, 0.18), (dwgu, Wg.grad, 0.18), (dwd, Wo.grad, 0.18)):
        assert rel(got, want) < limit, (rel(got, want), limit)
    # the same block serves fewer rows, without what training keeps; the same numbers, whatever the rows beside them
    serve = cfb.FfnSwigluFp8Block128(ctx, rows, H, F)
    y1 = torch.empty_like(y)
    serve.forward(x, r, gain, wgu, wd, y1)
    assert torch.equal(y1, y)
    # accumulation, and the same bits again
    dwgu2, dwd2, dg2, dx2 = dwgu.clone(), dwd.clone(), dg.clone(), torch.empty_like(dx)
    block.backward(dy, dh, gain, wgu, wd, dx2, dwgu2, dwd2, dg2, accumulate=True)
    assert torch.equal(dx2, dx) and torch.equal(dwgu2, dwgu + dwgu) and torch.equal(dwd2, dwd + dwd) and torch.equal(dg2, dg + dg)


def test_feed_forward_block_captured_while_another_stream_works(cfb, ctx):
    """Two blocks captured into graphs and replayed on two streams with new inputs in the same buffers: the bits of eager calls
    (the products share a context, but keep nothing in it)."""
    H, F = 512, 384
    w = [(cfb.Fp8Block128Weight(normal((2 * F, H), 80 + i, H ** -0.5)), cfb.Fp8Block128Weight(normal((H, F), 90 + i, F ** -0.5))) for i in range(2)]
    gain = normal((H,), 3)
    rows = (7, 300)
    blocks = [cfb.FfnSwigluFp8Block128(ctx, n, H, F, train=True) for n in rows]
    bufs = [[torch.empty((n, H), dtype=torch.bfloat16, device="cuda") for _ in range(4)] for n in rows]
    grads = [[torch.empty((2 * F, H), device="cuda"), torch.empty((H, F), device="cuda"), torch.empty(H, device="cuda")] for _ in rows]

    def step(i):
        x, y, dy, dx = bufs[i]
        blocks[i].forward(x, None, gain, *w[i], y)
        blocks[i].backward(dy, None, gain, *w[i], dx, *grads[i])

    def fill(seed):
        for i, n in enumerate(rows):
            bufs[i][0].copy_(normal((n, H), seed + i))
            bufs[i][2].copy_(normal((n, H), seed + 5 + i))

    def outputs(i):
        return [bufs[i][1].clone(), bufs[i][3].clone()] + [g.clone() for g in grads[i]]

    fill(100)
    streams, graphs = [torch.cuda.Stream() for _ in rows], []
    for i in range(2):
        streams[i].wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(streams[i]):
            step(i)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[i]):
            step(i)
        graphs.append(g)
    for seed in (200, 300):
        fill(seed)
        torch.cuda.synchronize()
        want = []
        for i in range(2):
            step(i)
            want.append(outputs(i))
        torch.cuda.synchronize()
        for i in range(2):
            for t in [bufs[i][1], bufs[i][3]] + grads[i]:
                t.zero_()
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                for _ in range(3):
                    graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, b) for a, b in zip(outputs(i), want[i]))
    ctx.poll_status()


def test_routed_experts_run(cfb, ctx):
    """Router, dispatch lists, permute of codes and descales, ragged products, SwiGLU, combine: the layer with block scales."""
    rows, H, F, E, k = 300, 256, 384, 5, 2
    x = normal((rows, H), 110)
    logits = torch.randn((rows, E), generator=gen(111), device="cuda")
    wgu = torch.stack([normal((2 * F, H), 120 + e, H ** -0.5) for e in range(E)])
    wd = torch.stack([normal((H, F), 130 + e, F ** -0.5) for e in range(E)])
    wgu8, dgu = torch.empty_like(wgu, dtype=torch.uint8), torch.empty((E, cdiv(2 * F, G), cdiv(H, G)), device="cuda")
    wd8, dd = torch.empty_like(wd, dtype=torch.uint8), torch.empty((E, cdiv(H, G), cdiv(F, G)), device="cuda")
    cfb.fp8_quantize_block128x128(wgu, wgu8, dgu)
    cfb.fp8_quantize_block128x128(wd, wd8, dd)
    T = rows * k
    counts, offsets = (torch.zeros(E, dtype=torch.int32, device="cuda") for _ in range(2))
    idx = torch.zeros((E, rows), dtype=torch.int32, device="cuda")
    rw = logits.clone()
    scratch = torch.empty(max(1, cfb.moe_route_dispatch_scratch_ints(rows, E)), dtype=torch.int32, device="cuda")
    cfb.moe_route_dispatch_lists(rw, rows, E, k, counts, offsets, idx, scratch)
    x8, dx = torch.empty((rows, H), dtype=torch.uint8, device="cuda"), torch.empty((rows, cdiv(H, G)), device="cuda")
    cfb.fp8_quantize_block128(x, x8, dx)
    xc, dxc = torch.empty((T, H), dtype=torch.uint8, device="cuda"), torch.empty((T, cdiv(H, G)), device="cuda")
    cfb.moe_gather_all_u8(x8, xc, idx, counts, offsets, rows, E, H)
    cfb.moe_gather_all_u8(dx.view(torch.uint8), dxc.view(torch.uint8), idx, counts, offsets, rows, E, 4 * cdiv(H, G))
    gu = torch.empty((T, 2 * F), dtype=torch.bfloat16, device="cuda")
    cfb.gemm_fp8_block128_nt_grouped(ctx, counts, offsets, xc, dxc, wgu8, dgu, gu)
    a8, da = torch.empty((T, F), dtype=torch.uint8, device="cuda"), cfb.block128_row_descale(T, F)
    cfb.swiglu_quantize_block128(gu[:, :F], gu[:, F:], a8, da)
    yc = torch.empty((T, H), dtype=torch.bfloat16, device="cuda")
    cfb.gemm_fp8_block128_nt_grouped(ctx, counts, offsets, a8, da, wd8, dd, yc)
    mixed = torch.empty((rows, H), dtype=torch.bfloat16, device="cuda")
    cfb.moe_combine_sorted_bf16(mixed, yc, rw, idx, counts, offsets, rows, E, H, accumulate=False)
    ctx.poll_status()
    assert int(counts.sum()) == T
    want = torch.zeros((rows, H), dtype=torch.float64, device="cuda")
    for e in range(E):
        o, n = int(offsets[e]), int(counts[e])
        at = idx[e, :n].long()
        assert torch.equal(xc[o:o + n], x8[at]) and torch.equal(dxc[o:o + n], dx[at])
        check_product(gu[o:o + n], value64(x8[at], dx[at], False, 1, G), value64(wgu8[e], dgu[e], False, G, G).t(), H)
        check_product(yc[o:o + n], value64(a8[o:o + n], da[o:o + n], False, 1, G), value64(wd8[e], dd[e], False, G, G).t(), F)
        want[at] += rw[at, e].double()[:, None] * yc[o:o + n].double()
    # one bf16 rounding per expert added (two of them): 2^-8 of the running sum each
    mag = torch.zeros_like(want)
    for e in range(E):
        o, n = int(offsets[e]), int(counts[e])
        at = idx[e, :n].long()
        mag[at] += (rw[at, e].double()[:, None] * yc[o:o + n].double()).abs()
    assert (mixed.double() - want).abs().le(k * 2.0 ** -8 * (1 + 2.0 ** -6) * mag + 1e-30).all()


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_calls_back_to_back_are_ordered(cfb, ctx, rows):
    """Each kernel may be scheduled while the one before it drains: a chain of small calls that overwrite each other's inputs gives
    the same bits as the same calls with the GPU idle in between, eagerly and replayed from a graph."""
    H, F = 256, 384
    wgu = cfb.Fp8Block128Weight(normal((2 * F, H), 901, 0.05))
    wd = cfb.Fp8Block128Weight(normal((H, F), 902, 0.05))
    gain, x0, dy0 = normal((H,), 903), normal((rows, H), 904), normal((rows, H), 905, 1e-2)
    ffn = cfb.FfnSwigluFp8Block128(ctx, rows, H, F, train=True)
    x, dy, dx = torch.empty_like(x0), torch.empty_like(dy0), torch.empty_like(x0)
    dgu, dd = torch.empty((2 * F, H), device="cuda"), torch.empty((H, F), device="cuda")
    dgain = torch.empty(H, device="cuda")
    state = (x, ffn.h, dx, dgu, dd, dgain)

    def layers(idle):
        x.copy_(x0)
        dy.copy_(dy0)
        dgain.zero_(), dgu.zero_(), dd.zero_()
        for i in range(6):
            ffn.forward(x, ffn.h if i else None, gain, wgu, wd, x)
            idle()
            ffn.backward(dy, dy, gain, wgu, wd, dy, dgu, dd, dgain, accumulate=True)
            idle()
            cfb.fp8_quantize_block128(x, *ffn.n8)
            cfb.add_rmsnorm_quantize_block128(x, None, gain, None, None, x, *ffn.n8)
            idle()
        dx.copy_(dy)

    layers(torch.cuda.synchronize)
    want = [t.clone() for t in state]
    assert all(torch.isfinite(t).all() for t in want)
    for _ in range(5):
        layers(lambda: None)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(state, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layers(lambda: None)
    for _ in range(5):
        for t in state:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(state, want))
    ctx.poll_status()
