"""What the block-scaled FP8 operators have to do, at real sizes: cases, inputs, plain forms and 64-bit definitions.

FP8 codes come with one float32 factor ("descale") for every group of 128 neighbouring values: value = code * descale.
Three operators work on that format:

  quantize  bf16 -> codes + descales, with the groups along the rows (1x128, operands contracted along a row), along the
            columns (128x1, operands contracted over tokens), both from one read, or in 128x128 blocks (weights); from a
            matrix, from silu(gate) * up, or from the gradient of silu(gate) * up
  norm      h = x + residual, RMS norm of h, codes + descales of the normalised row; and the gradient
  matmul    C[m,n] = sum over blocks b of da[m,b] * db[n,b] * sum over k in b of A[m,k] * B[n,k]: forward (nt), with ragged
            expert groups (grouped), data gradient (nn) and weight gradient (dw)

`own = False` computes them with elementary torch operations in float32; `own = True` calls the framework.
"""
import importlib
import math

import numpy as np
import torch

own = False

G = 128                                         # values that share a scale
MAXIMA = {"e4m3": 448.0, "e5m2": 57344.0}
TYPES = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
EPS = 1e-6


def cdiv(a, b):
    return -(-a // b)


def pad16(n):
    return cdiv(n, 16) * 16


# ---------------------------------------------------------------- cases
def listed():
    return [
        # the gradient that arrives at a linear layer in training: codes for the data gradient and for the weight gradient
        {"name": "quantize_grad_both", "op": "quantize", "form": "both", "fmt": "e5m2", "rows": 8192, "cols": 4096},
        # between gate/up and down projection of one prompt of odd length, gate and up as halves of one matrix
        {"name": "quantize_swiglu_prompt", "op": "quantize", "form": "swiglu", "fmt": "e4m3", "rows": 2039, "cols": 14336},
        # the same place in the backward pass of training: gradients of gate and up, coded for both products behind it
        {"name": "quantize_swiglu_grad", "op": "quantize", "form": "swiglu_grad", "fmt": "e4m3", "rows": 4096, "cols": 14336},
        # one token being decoded: latency
        {"name": "norm_one_token", "op": "norm", "form": "forward", "rows": 1, "cols": 4096},
        # a large prefill or training batch
        {"name": "norm_batch", "op": "norm", "form": "forward", "rows": 16384, "cols": 4096},
        {"name": "norm_grad", "op": "norm", "form": "backward", "rows": 8192, "cols": 4096},
        # gate/up projection while four sequences are decoded: the weights are read once
        {"name": "matmul_decode", "op": "matmul", "form": "nt", "fmt": "e4m3", "M": 4, "N": 28672, "K": 4096},
        # a prompt of odd length through a layer whose sizes are no multiples of the tiles or of 128
        {"name": "matmul_odd", "op": "matmul", "form": "nt", "fmt": "e4m3", "M": 1531, "N": 4104, "K": 5416},
        # gate/up projection of a training batch: the largest
        {"name": "matmul_batch", "op": "matmul", "form": "nt", "fmt": "e4m3", "M": 16384, "N": 28672, "K": 4096},
        # down projection of eight experts, ragged, one expert idle
        {"name": "matmul_experts", "op": "matmul", "form": "grouped", "fmt": "e4m3", "M": 4096, "N": 4096, "K": 14336, "E": 8},
        # data and weight gradient of a projection
        {"name": "matmul_data_grad", "op": "matmul", "form": "nn", "fmt": "e5m2", "M": 8192, "N": 4096, "K": 14336},
        {"name": "matmul_weight_grad", "op": "matmul", "form": "dw", "fmt": "e5m2", "M": 4096, "N": 14336, "K": 8192},
    ]


def _spread(rng, lo, hi, step=1):
    """A number between lo and hi, even over the logarithm, a multiple of step."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi, max(lo, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(["quantize", "norm", "matmul", "matmul"])
    if op == "quantize":
        form = rng.choice(["row", "col", "both", "block", "swiglu", "swiglu_grad"])
        # the two halves of a SwiGLU gradient lie side by side: each a multiple of the group
        cols = _spread(rng, 256, 14336, 128 if form == "swiglu_grad" else rng.choice([1, 8, 128]))
        rows = _spread(rng, 1, min(32768, (1 << 27) // cols))
        fmt = "e4m3" if form in ("block", "swiglu") else rng.choice(["e4m3", "e5m2"])
        return {"op": op, "form": form, "fmt": fmt, "rows": rows, "cols": cols}
    if op == "norm":
        form = rng.choice(["forward", "forward", "backward"])
        cols = _spread(rng, 512, 16384, rng.choice([1, 8, 128, 512]))
        return {"op": op, "form": form, "rows": _spread(rng, 1, min(32768, (1 << 26) // cols)), "cols": cols}
    form = rng.choice(["nt", "nt", "nt", "grouped", "nn", "dw"])
    step = rng.choice([1, 8, 128])
    N, K = _spread(rng, 256, 16384, step), _spread(rng, 256, 16384, step)
    most = min(16384, int(4e11 / N / K))
    case = {"op": op, "form": form, "fmt": "e4m3", "M": _spread(rng, 1, max(1, most)), "N": N, "K": K}
    if form == "nn":
        case |= {"fmt": rng.choice(["e4m3", "e5m2"]), "N": pad16(N)}
    if form == "dw":
        case |= {"fmt": rng.choice(["e4m3", "e5m2"]), "M": _spread(rng, 256, 8192, 16), "N": pad16(N), "K": max(1, min(16384, int(4e11 / N / 8192)))}
        case["K"] = _spread(rng, 1, max(2, case["K"]))
    if form == "grouped":
        case |= {"E": rng.randint(2, 16)}
        case |= {"M": max(1, min(8192, case["M"] // case["E"]))}
    return case


def work(case):
    if case["op"] == "quantize":
        n = case["rows"] * case["cols"]
        reads = {"swiglu": 4, "swiglu_grad": 6}.get(case["form"], 2)
        writes = {"both": 2, "swiglu_grad": 4}.get(case["form"], 1)
        flops = {"swiglu": 8, "swiglu_grad": 18}.get(case["form"], 2)
        groups = {"block": 1 / (G * G)}.get(case["form"], writes / G)
        return {"bytes": n * (reads + writes + 4 * groups), "flops": n * flops}
    if case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        if case["form"] == "forward":
            return {"bytes": rows * cols * (2 + 2 + 2 + 1 + 4 / G) + 2 * cols + 4 * rows, "flops": rows * cols * 8}
        return {"bytes": rows * cols * (2 + 2 + 2 + 2) + 6 * cols + 4 * rows, "flops": rows * cols * 11}
    M, N, K, form = case["M"], case["N"], case["K"], case["form"]
    weights = N * K * case.get("E", 1)
    out = 4 if form == "dw" else 2
    scales = 4 * (M + N) * cdiv(K, G) if form == "dw" else 4 * (M * cdiv(K, G) + weights / (G * G))
    return {"bytes": M * K + weights + scales + out * M * N, "flops": 2 * M * N * K}


# ---------------------------------------------------------------- inputs
def _normal(gen, shape, std=1.0, outliers=0.0):
    x = torch.randn(shape, generator=gen, device="cuda") * std
    if outliers:
        x = torch.where(torch.rand(shape, generator=gen, device="cuda") < outliers, x * 20.0, x)
    return x.to(torch.bfloat16)


def _coded(x, fmt, rows_per, cols_per):
    """Codes (uint8, row pitch a multiple of 16 bytes) and descales of a bf16 matrix or a stack of them."""
    q, d = _quantize(x.float(), fmt, rows_per, cols_per)
    R, C = x.shape[-2:]
    buf = torch.zeros((*x.shape[:-1], pad16(C)), dtype=torch.uint8, device="cuda")
    buf[..., :C] = q.view(torch.uint8)
    return buf[..., :C], d


def _outputs(case):
    """The buffers a program keeps for the results."""
    def codes(r, c):
        return torch.zeros((r, pad16(c)), dtype=torch.uint8, device="cuda")[:, :c]

    def rowd(r, c):          # [rows, groups], the rows next to each other in memory
        return torch.zeros((cdiv(c, G), r), dtype=torch.float32, device="cuda").t()

    def cold(r, c):
        return torch.zeros((cdiv(r, G), c), dtype=torch.float32, device="cuda")

    if case["op"] == "quantize":
        R, C, form = case["rows"], case["cols"] * (2 if case["form"] == "swiglu_grad" else 1), case["form"]
        if form == "block":
            return {"q": codes(R, C), "d": torch.zeros((cdiv(R, G), cdiv(C, G)), device="cuda")}
        o = {}
        if form != "col":
            o |= {"q": codes(R, C), "d": rowd(R, C)}
        if form in ("col", "both", "swiglu_grad"):
            o |= {"qc": codes(R, C), "dc": cold(R, C)}
        return o
    if case["op"] == "norm":
        R, C = case["rows"], case["cols"]
        if case["form"] == "forward":
            return {"h": torch.empty((R, C), dtype=torch.bfloat16, device="cuda"), "rms": torch.empty(R, device="cuda"),
                    "q": codes(R, C), "d": rowd(R, C)}
        return {"dx": torch.empty((R, C), dtype=torch.bfloat16, device="cuda"), "dg": torch.empty(C, device="cuda")}
    return {"c": torch.zeros((case["M"], case["N"]), dtype=torch.float32 if case["form"] == "dw" else torch.bfloat16, device="cuda")}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": dict(case), "o": _outputs(case)}
    if case["op"] == "quantize":
        R, C, form = case["rows"], case["cols"], case["form"]
        if form in ("swiglu", "swiglu_grad"):
            gu = _normal(gen, (R, 2 * C), 1.0, 0.001)
            s |= {"gate": gu[:, :C], "up": gu[:, C:]}
            if form == "swiglu_grad":
                s["dh"] = _normal(gen, (R, C), 1e-3, 0.001)
        else:
            s["x"] = _normal(gen, (R, C), 0.02 if form == "block" else 1e-3 if case["fmt"] == "e5m2" else 1.0, 0.0 if form == "block" else 0.001)
    elif case["op"] == "norm":
        R, C = case["rows"], case["cols"]
        s["g"] = (1.0 + 0.1 * torch.randn(C, generator=gen, device="cuda")).to(torch.bfloat16)
        if case["form"] == "forward":
            s |= {"x": _normal(gen, (R, C), 1.0, 0.001), "r": _normal(gen, (R, C), 2.0, 0.001)}
        else:
            s |= {"dy": _normal(gen, (R, C), 1e-2), "h": _normal(gen, (R, C), 2.0, 0.001), "dh": _normal(gen, (R, C), 1e-2)}
            s["rms"] = (s["h"].double().square().mean(1) + EPS).sqrt().float()
    else:
        M, N, K, form = case["M"], case["N"], case["K"], case["form"]
        if form == "nt":
            s["a"], s["da"] = _coded(_normal(gen, (M, K), 1.0, 0.001), "e4m3", 1, G)
            s["b"], s["db"] = _coded(_normal(gen, (N, K), 0.02), "e4m3", G, G)
        elif form == "grouped":
            E = case["E"]
            s["a"], s["da"] = _coded(_normal(gen, (M, K), 1.0, 0.001), "e4m3", 1, G)
            s["b"], s["db"] = _coded(_normal(gen, (E, N, pad16(K)), 0.02)[..., :K], "e4m3", G, G)
            # popularity falls with the expert's number, the second one idle, a few rows behind the last group
            share = np.arange(1, E + 1, dtype=np.float64) ** -1.1 * (1.0 + 0.1 * (int(seed) % 3))
            share[1] = 0.0
            counts = np.floor((M - min(3, M - 1)) * share / share.sum()).astype(np.int32)
            s["counts"] = torch.from_numpy(counts).cuda()
            s["offsets"] = torch.from_numpy((np.cumsum(counts) - counts).astype(np.int32)).cuda()
        elif form == "nn":
            s["a"], s["da"] = _coded(_normal(gen, (M, K), 1e-3, 0.001), case["fmt"], 1, G)
            s["b"], s["db"] = _coded(_normal(gen, (K, N), 0.02), "e4m3", G, G)
        else:
            s["a"], s["da"] = _coded(_normal(gen, (K, M), 1.0, 0.001), "e4m3", G, 1)
            s["b"], s["db"] = _coded(_normal(gen, (K, N), 1e-3, 0.001), case["fmt"], G, 1)
        if form in ("nt", "grouped", "nn"):
            s["da"] = s["da"].t().contiguous().t()          # the rows next to each other in memory, as the quantiser leaves them
    return s


# ---------------------------------------------------------------- plain forms
def _tiles(x, rows_per, cols_per):
    """[..., R, C] -> [..., blocks of rows, rows_per, blocks of columns, cols_per], zeros behind the edges."""
    R, C = x.shape[-2:]
    x = torch.nn.functional.pad(x, (0, -C % cols_per, 0, -R % rows_per))
    return x.reshape(*x.shape[:-2], x.shape[-2] // rows_per, rows_per, x.shape[-1] // cols_per, cols_per)


def _quantize(x, fmt, rows_per, cols_per):
    R, C = x.shape[-2:]
    t = _tiles(x, rows_per, cols_per)
    a = t.abs().amax(dim=(-3, -1), keepdim=True).clamp(min=1e-12)
    q = (t * (MAXIMA[fmt] / a)).clamp(-MAXIMA[fmt], MAXIMA[fmt]).to(TYPES[fmt])
    q = q.reshape(*x.shape[:-2], t.shape[-4] * rows_per, t.shape[-2] * cols_per)[..., :R, :C]
    d = (a / MAXIMA[fmt]).squeeze(-1).squeeze(-2)
    return q.contiguous(), d.contiguous()


def _values(codes, d, fmt, rows_per, cols_per):
    R, C = codes.shape[-2:]
    d = d.repeat_interleave(rows_per, -2)[..., :R, :] if rows_per > 1 else d
    d = d.repeat_interleave(cols_per, -1)[..., :C] if cols_per > 1 else d
    return codes.contiguous().view(TYPES[fmt]).float() * d


def _source(s):
    form = s["case"]["form"]
    if form not in ("swiglu", "swiglu_grad"):
        return s["x"].float()
    g, u = s["gate"].float(), s["up"].float()
    sig = 1.0 / (1.0 + torch.exp(-g))
    if form == "swiglu":
        return g * sig * u
    dh = s["dh"].float()
    return torch.cat([dh * u * sig * (1.0 + g * (1.0 - sig)), dh * g * sig], dim=1)


def _plain(s):
    case, form = s["case"], s["case"]["form"]
    if case["op"] == "quantize":
        x, o = _source(s), {}
        if form == "block":
            q, d = _quantize(x, case["fmt"], G, G)
            return {"q": q, "d": d}
        if form != "col":
            o["q"], o["d"] = _quantize(x, case["fmt"], 1, G)
        if form in ("col", "both", "swiglu_grad"):
            o["qc"], o["dc"] = _quantize(x, case["fmt"], G, 1)
        return o
    if case["op"] == "norm":
        g = s["g"].float()
        if form == "forward":
            h = (s["x"].float() + s["r"].float()).to(torch.bfloat16)
            hf = h.float()
            rms = (hf.square().mean(1) + EPS).sqrt()
            q, d = _quantize(hf / rms[:, None] * g, "e4m3", 1, G)
            return {"h": h, "rms": rms, "q": q, "d": d}
        dy, xhat = s["dy"].float(), s["h"].float() / s["rms"][:, None]
        u = dy * g
        dx = (u - xhat * (u * xhat).mean(1, keepdim=True)) / s["rms"][:, None] + s["dh"].float()
        return {"dx": dx.to(torch.bfloat16), "dg": (dy * xhat).sum(0, dtype=torch.float64).float()}
    if form == "nt":
        return {"c": (_values(s["a"], s["da"], "e4m3", 1, G) @ _values(s["b"], s["db"], "e4m3", G, G).t()).to(torch.bfloat16)}
    if form == "grouped":
        row = torch.arange(case["M"], device="cuda")
        ends = torch.cumsum(s["counts"], 0)
        expert = torch.searchsorted(ends, row, right=True)
        every = _values(s["a"], s["da"], "e4m3", 1, G)[None] @ _values(s["b"], s["db"], "e4m3", G, G).transpose(1, 2)
        picked = every[expert.clamp(max=case["E"] - 1), row].to(torch.bfloat16)
        return {"c": torch.where((row < ends[-1])[:, None], picked, s["o"]["c"])}
    if form == "nn":
        return {"c": (_values(s["a"], s["da"], case["fmt"], 1, G) @ _values(s["b"], s["db"], "e4m3", G, G)).to(torch.bfloat16)}
    return {"c": _values(s["a"], s["da"], "e4m3", G, 1).t() @ _values(s["b"], s["db"], case["fmt"], G, 1)}


# ---------------------------------------------------------------- the framework's calls
_kept = {}


def _framework():
    """The package and the context a program creates once."""
    if not _kept:
        cfb = importlib.import_module("canopy-foundry_b200")
        _kept["ops"], _kept["ctx"] = cfb, cfb.Fp8Ctx()
    return _kept["ops"], _kept["ctx"]


def _own(s):
    cfb, ctx = _framework()
    case, form, o = s["case"], s["case"]["form"], s["o"]
    e5m2 = case.get("fmt") == "e5m2"
    if case["op"] == "quantize":
        if form == "block":
            cfb.fp8_quantize_block128x128(s["x"], o["q"], o["d"])
        elif form == "swiglu":
            cfb.swiglu_quantize_block128(s["gate"], s["up"], row8=o["q"], row_descale=o["d"])
        elif form == "swiglu_grad":
            cfb.swiglu_backward_quantize_block128(s["gate"], s["up"], s["dh"], row8=o["q"], row_descale=o["d"], col8=o["qc"],
                                                  col_descale=o["dc"], is_e5m2=e5m2)
        else:
            cfb.fp8_quantize_block128(s["x"], row8=o.get("q"), row_descale=o.get("d"), col8=o.get("qc"), col_descale=o.get("dc"),
                                      is_e5m2=e5m2)
        return {k: v.view(TYPES[case["fmt"]]) if k in ("q", "qc") else v for k, v in o.items()}
    if case["op"] == "norm":
        if form == "forward":
            cfb.add_rmsnorm_quantize_block128(s["x"], s["r"], s["g"], o["h"], o["rms"], out8=o["q"], descale=o["d"], eps=EPS)
            return o | {"q": o["q"].view(TYPES["e4m3"])}
        if "scratch" not in s:
            s["scratch"] = torch.empty(cfb.add_rmsnorm_backward_scratch_floats(*s["h"].shape), device="cuda")
        cfb.add_rmsnorm_backward(s["dy"], s["h"], s["g"], s["rms"], s["dh"], o["dx"], o["dg"], s["scratch"])
        return o
    if form == "nt":
        cfb.gemm_fp8_block128_nt(ctx, s["a"], s["da"], s["b"], s["db"], o["c"])
    elif form == "grouped":
        cfb.gemm_fp8_block128_nt_grouped(ctx, s["counts"], s["offsets"], s["a"], s["da"], s["b"], s["db"], o["c"])
    elif form == "nn":
        cfb.gemm_fp8_block128_nn(ctx, s["a"], s["da"], s["b"], s["db"], o["c"], a_is_e5m2=e5m2)
    else:
        cfb.gemm_fp8_block128_dw(ctx, s["a"], s["da"], s["b"], s["db"], o["c"], dy_is_e5m2=e5m2)
    return o


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------- the definitions in 64 bits
def _table(fmt):
    """Value of each of the 256 codes, from the format's definition: sign, exponent and mantissa bits, bias."""
    mant, bias = (3, 7) if fmt == "e4m3" else (2, 15)
    code = np.arange(256)
    m, e = code & ((1 << mant) - 1), (code & 0x7f) >> mant
    v = np.where(e == 0, m * 2.0 ** (1 - bias - mant), (1.0 + m * 2.0 ** -mant) * 2.0 ** (e - bias))
    return torch.from_numpy(np.where(code & 0x80, -v, v)).cuda()


def _nearest(v, fmt):
    """v (64 bits) rounded to the format's values, ties to even; the largest finite value where v is beyond it."""
    mant, low = (3, -6) if fmt == "e4m3" else (2, -14)
    _, e = torch.frexp(v)                          # |v| in [2^(e-1), 2^e)
    step = torch.ldexp(torch.ones_like(v), torch.clamp(e - 1, min=low) - mant)
    return torch.clamp(torch.round(v / step) * step, -MAXIMA[fmt], MAXIMA[fmt])


def _groups64(v, fmt, along):
    """Codes' values and descales of v with groups of 128 along dimension `along`, one group after the other."""
    qs, ds = [], []
    for part in torch.split(v, G, dim=along):
        a = part.abs().max(dim=along, keepdim=True).values.clamp(min=1e-12)
        qs.append(_nearest(part / a * MAXIMA[fmt], fmt))
        ds.append(a / MAXIMA[fmt])
    return torch.cat(qs, along), torch.cat(ds, along)


def exact(case, seed):
    s = prepare(case, seed)
    form, fmt = case["form"], case.get("fmt", "e4m3")
    if case["op"] == "quantize":
        if form == "block":
            rows = [_block64(p, fmt) for p in torch.split(s["x"].double(), G, dim=0)]
            return {"q": torch.cat([q for q, _ in rows]), "d": torch.cat([d for _, d in rows])}
        if form in ("swiglu", "swiglu_grad"):
            g, u = s["gate"].double(), s["up"].double()
            silu, sig = g * torch.sigmoid(g), torch.sigmoid(g)
            v = silu * u if form == "swiglu" else torch.cat([s["dh"].double() * u * (sig + silu * (1 - sig)), s["dh"].double() * silu], 1)
        else:
            v = s["x"].double()
        o = {}
        if form != "col":
            o["q"], o["d"] = _groups64(v, fmt, 1)
        if form in ("col", "both", "swiglu_grad"):
            o["qc"], o["dc"] = _groups64(v, fmt, 0)
        return o
    if case["op"] == "norm":
        g = s["g"].double()
        if form == "forward":
            h = (s["x"].double() + s["r"].double()).to(torch.bfloat16)      # the stream itself is held in bf16
            rms = (h.double().pow(2).sum(1) / case["cols"] + EPS).sqrt()
            q, d = _groups64(h.double() * g / rms[:, None], "e4m3", 1)
            return {"h": h.double(), "rms": rms, "q": q, "d": d}
        r = 1.0 / s["rms"].double()[:, None]
        u, h = s["dy"].double() * g, s["h"].double()
        dot = (u * h).sum(1, keepdim=True)
        return {"dx": s["dh"].double() + r * u - r ** 3 * h * dot / case["cols"], "dg": (s["dy"].double() * h * r).sum(0)}
    # products: block after block of the contraction, the descales applied to each block's sum
    K = case["K"]
    a = _table("e4m3" if form in ("nt", "grouped", "dw") else fmt)[s["a"].long()]
    tb = _table(fmt if form == "dw" else "e4m3")
    if form == "dw":
        b, c = tb[s["b"].long()], 0.0
        for i in range(cdiv(K, G)):
            k = slice(i * G, min(K, (i + 1) * G))
            c = c + (a[k].t() @ b[k]) * s["da"][i].double()[:, None] * s["db"][i].double()[None]
        return {"c": c}
    c = s["o"]["c"].double()
    spans = [(0, case["M"])] if form != "grouped" else list(zip(s["offsets"].tolist(), s["counts"].tolist()))
    for e, (first, rows) in enumerate(spans):
        if rows == 0:
            continue
        b = tb[(s["b"][e] if form == "grouped" else s["b"]).long()]
        db = (s["db"][e] if form == "grouped" else s["db"]).double()
        if form == "nn":
            b, db = b.t(), db.t()
        at, acc = slice(first, first + rows), 0.0
        for i in range(cdiv(K, G)):
            k = slice(i * G, min(K, (i + 1) * G))
            per_n = db[:, i].repeat_interleave(G)[: case["N"]]
            acc = acc + (a[at, k] @ b[:, k].t()) * s["da"][at, i].double()[:, None] * per_n[None]
        c[at] = acc
    return {"c": c}


def _block64(rows, fmt):
    qs, ds = [], []
    for part in torch.split(rows, G, dim=1):
        a = part.abs().max().clamp(min=1e-12)
        qs.append(_nearest(part / a * MAXIMA[fmt], fmt))
        ds.append((a / MAXIMA[fmt]).reshape(1, 1))
    return torch.cat(qs, 1), torch.cat(ds, 1)
