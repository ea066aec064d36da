// Block-scaled FP8 quantiser: one fp32 scale for every group of 128 values.
//
//   a = max(max|v| over the group, 1e-12),  descale = a / FMAX,  code = fp8(v * FMAX / a)      FMAX = 448 or 57344
//
// Groups run along a row (1x128: operands whose contraction runs along the row), down a column (128x1: operands of the
// weight gradient, contracted over tokens) or are 128x128 blocks (weights). v is a bf16 matrix, silu(gate) * up, or the
// gradient of silu(gate) * up. Products and amax are taken in fp32 and rounded ONCE, to the code: the descale is held in
// 32 bits, and no bf16 rounding lies between the activation and its code.
// The reference scales per tensor only; the formulas generalise kernels/fp8.cu:34-49 to groups.
//
// All forms are streams: they are bound by the bytes of inputs and codes (2 B in + 1 B out per element and output of the
// plain form), so every input element is read once whatever the number of outputs. A block owns a tile of 128 columns;
// a half-warp reads 128 columns of one row (256 contiguous bytes) and holds that row's group, so the row amax is four
// shuffles; the column amax meets in shared memory across the rows of the tile; the values stay in registers in between.
// Like the norm and the products these kernels, but for the one for weights, may be scheduled while the kernel before them drains, and
// wait for it before they touch memory: a feed-forward layer of one token (4096 / 14336, four launches) takes 39.9 us instead of 43.1.
#include <atomic>
#include <cfloat>

#include "cf_common.cuh"
#include "cf_internal.cuh"

namespace cf {
namespace {

constexpr int G = 128;                       // values per scale
constexpr float kFloorAmax = 1e-12f;

enum Src { SRC_PLAIN = 0, SRC_SWIGLU = 1, SRC_SWIGLU_GRAD = 2 };

struct QuantParams {
    const uint16_t* x;        // plain source, or gate
    const uint16_t* up;
    const uint16_t* dh;
    long long ld_x;           // row pitch of x / gate / up in elements
    long long ld_dh;
    int rows, cols;           // of the source
    uint8_t* row8;
    long long ld_row8;
    float* row_d;
    long long rd_row, rd_blk; // strides of the row descales
    uint8_t* col8;
    long long ld_col8;
    float* col_d;
    long long cd_blk, cd_col; // strides of the column descales
    int col_blocks;
    int vec_in, vec_row8, vec_col8;
};

__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
    f[0] = __uint_as_float(v.x << 16); f[1] = __uint_as_float(v.x & 0xffff0000u);
    f[2] = __uint_as_float(v.y << 16); f[3] = __uint_as_float(v.y & 0xffff0000u);
    f[4] = __uint_as_float(v.z << 16); f[5] = __uint_as_float(v.z & 0xffff0000u);
    f[6] = __uint_as_float(v.w << 16); f[7] = __uint_as_float(v.w & 0xffff0000u);
}
// Eight bf16 values of a row as one 16-byte load, or element by element where the row's base or its end forbid that. Plain loads:
// read-only ones could be moved ahead of the wait for the grid that writes them.
__device__ __forceinline__ uint4 load8(const uint16_t* p, int n, bool vec) {
    if (vec && n >= 8) return *reinterpret_cast<const uint4*>(p);
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e < n) w[e >> 1] |= static_cast<uint32_t>(p[e]) << (16 * (e & 1));
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void store8(uint8_t* p, const uint2& q, int n, bool vec) {
    if (vec && n >= 8) { *reinterpret_cast<uint2*>(p) = q; return; }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e < n) p[e] = static_cast<uint8_t>((e < 4 ? q.x >> (8 * e) : q.y >> (8 * (e - 4))) & 0xffu);
}
// FMAX / a in two parts: `hi` with 16 significant bits, `lo` the rest to 40 bits. For a bf16 value v (8 bits) v * hi is exact and
// fma(v, lo, v * hi) the correctly rounded v * FMAX / a, exact where that is representable. That matters: quotients of bf16
// numbers land exactly between two codes about once in three hundred values (ties go to the even code), and with one rounded
// factor such a value falls to either side. Price: 15 % of both groupings of 8192 x 4096, 32.5 us (67 to 70 % of the issue
// slots; its 136 MB take 20.8).
struct Scale2 { float hi, lo; };
__device__ __forceinline__ Scale2 scale2(float fmax, float a) {
    const float s = __fdiv_rn(fmax, a);
    const float hi = __uint_as_float(__float_as_uint(s) & 0xffffff00u);
    const float rest = fmaf(-s, a, fmax);                    // exact: what the rounded quotient leaves
    const float lo = fmaf(rest, s * (1.0f / fmax), s - hi);
    return {hi, isfinite(lo) ? lo : 0.0f};                   // a group with an infinity: s is 0
}
template <bool E5M2>
__device__ __forceinline__ uint2 code8x(const float (&f)[8], float hi, float lo) {
    float q[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = fmaf(f[e], lo, f[e] * hi);
    return make_uint2(cvt_fp8x4<E5M2>(q[0], q[1], q[2], q[3]), cvt_fp8x4<E5M2>(q[4], q[5], q[6], q[7]));
}
template <bool E5M2>
__device__ __forceinline__ uint2 code8(const float (&f)[8], float s) {
    return make_uint2(cvt_fp8x4<E5M2>(f[0] * s, f[1] * s, f[2] * s, f[3] * s), cvt_fp8x4<E5M2>(f[4] * s, f[5] * s, f[6] * s, f[7] * s));
}
template <bool E5M2>
__device__ __forceinline__ uint2 code8c(const float (&f)[8], const float (&s)[8]) {
    return make_uint2(cvt_fp8x4<E5M2>(f[0] * s[0], f[1] * s[1], f[2] * s[2], f[3] * s[3]),
                      cvt_fp8x4<E5M2>(f[4] * s[4], f[5] * s[5], f[6] * s[6], f[7] * s[7]));
}
__device__ __forceinline__ float half_warp_max(float v) {
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
    return v;
}
// Maxima of two packed bf16 values (non-negative ones here); a NaN yields to the other operand, like fmaxf.
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// Reciprocal good to one unit in the last place, one instruction. A Newton step on it, or on a quotient's remainder taken with a
// fused multiply-add (P. W. Markstein, Computation of elementary functions on the IBM RISC System/6000 processor, IBM J. Res. Dev.
// 34, 1990), squares the error: what is left before the last rounding is below 2^-44, so the result is the rounded quotient but for
// values that close to the middle of two numbers.
__device__ __forceinline__ float rcp(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// silu(g) * u = g / (1 + exp(-g)) * u, with the sum held down to the largest finite number: for g below -87.3 the reciprocal then
// is zero and so is silu, which is less than 2^-119 there (g multiplies what is left of the sigmoid, so a cut of the exponent
// alone would leave a value that grows with |g|). The quotient q of an infinite g is held down in the correction only: the correction
// is then infinite too, of the same sign, instead of the NaN of inf - inf. NaN, and -inf (inf * 0), give NaN.
__device__ __forceinline__ float swiglu(float g, float u) {
    const float d = 1.0f + fminf(expf(-g), FLT_MAX), r = rcp(d);
    const float q = g * r;
    return fmaf(fmaf(-d, fminf(q, FLT_MAX), g), r, q) * u;
}

// Values of a tile as the emitter wants them: RPT rows x 8 columns per thread. Bf16 sources stay packed (the row is unpacked
// twice, which is cheaper than the registers); computed ones are fp32.
template <int RPT>
struct PackedTile {
    uint4 v[RPT];
    __device__ __forceinline__ void row(int i, float (&f)[8]) const { unpack8(v[i], f); }
};
template <int RPT>
struct FloatTile {
    float v[RPT][8];
    __device__ __forceinline__ void row(int i, float (&f)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = v[i][e];
    }
};

template <class T>
struct IsPacked { static constexpr bool value = false; };
template <int RPT>
struct IsPacked<PackedTile<RPT>> { static constexpr bool value = true; };

// Codes and descales of a tile: row i of the thread at r0 + rg + i * RG, columns c0 + 8 cg. `shift`: where the outputs' columns
// start (the second half of the SwiGLU gradient lies behind the first).
template <int T, int RPT, bool ROW, bool COL, bool E5M2, class Tile>
__device__ __forceinline__ void emit_tile(const QuantParams& p, const Tile& t, int r0, int c0, int shift, float* s_col) {
    constexpr int RG = T / 16;
    constexpr float FMAX = E5M2 ? 57344.0f : 448.0f;
    const int cg = threadIdx.x & 15, rg = threadIdx.x >> 4, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int col = c0 + cg * 8;
    const int n = min(8, p.cols - col);
    float amax[RPT];               // of each row's group
    float cmax[8];                 // of each column over this warp's rows
    if constexpr (IsPacked<Tile>::value) {
        uint32_t rm[(RPT + 1) / 2], cm[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            const uint32_t w[4] = {t.v[i].x & 0x7fff7fffu, t.v[i].y & 0x7fff7fffu, t.v[i].z & 0x7fff7fffu, t.v[i].w & 0x7fff7fffu};
            if (COL) {
#pragma unroll
                for (int q = 0; q < 4; ++q) cm[q] = max2(cm[q], w[q]);
            }
            if (ROW) {             // two rows share a register on their way through the half-warp
                const uint32_t m = max2(max2(w[0], w[1]), max2(w[2], w[3]));
                const uint32_t one = max2(m, m >> 16) & 0xffffu;
                rm[i >> 1] = (i & 1) ? rm[i >> 1] | (one << 16) : one;
            }
        }
        if (ROW) {
#pragma unroll
            for (int h = 0; h < (RPT + 1) / 2; ++h) {
#pragma unroll
                for (int off = 8; off > 0; off >>= 1) rm[h] = max2(rm[h], __shfl_xor_sync(0xffffffffu, rm[h], off));
            }
#pragma unroll
            for (int i = 0; i < RPT; ++i) amax[i] = __uint_as_float((i & 1) ? rm[i >> 1] & 0xffff0000u : rm[i >> 1] << 16);
        }
        if (COL) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                cm[q] = max2(cm[q], __shfl_xor_sync(0xffffffffu, cm[q], 16));
                cmax[2 * q] = __uint_as_float(cm[q] << 16);
                cmax[2 * q + 1] = __uint_as_float(cm[q] & 0xffff0000u);
            }
        }
    } else {
        if (ROW) {
#pragma unroll
            for (int i = 0; i < RPT; ++i) {
                float a = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) a = fmaxf(a, fabsf(t.v[i][e]));
                amax[i] = half_warp_max(a);
            }
        }
        if (COL) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                cmax[e] = 0.0f;
#pragma unroll
                for (int i = 0; i < RPT; ++i) cmax[e] = fmaxf(cmax[e], fabsf(t.v[i][e]));
                cmax[e] = fmaxf(cmax[e], __shfl_xor_sync(0xffffffffu, cmax[e], 16));
            }
        }
    }
    if (COL && lane < 16) {
        float4* d = reinterpret_cast<float4*>(s_col + warp * G + cg * 8);
        d[0] = make_float4(cmax[0], cmax[1], cmax[2], cmax[3]);
        d[1] = make_float4(cmax[4], cmax[5], cmax[6], cmax[7]);
    }
    if (ROW) {
        // lane cg of a half-warp divides for row cg (of RPT), the quotients are handed round: one pair of divisions per
        // thread instead of one per row
        float mine = amax[0];
#pragma unroll
        for (int i = 1; i < RPT; ++i)
            if (cg == i) mine = amax[i];
        mine = fmaxf(mine, kFloorAmax);
        Scale2 scale;
        if constexpr (IsPacked<Tile>::value) scale = scale2(FMAX, mine);
        else scale = {__fdiv_rn(FMAX, mine), 0.0f};         // computed values: no exact quotient to keep
        const int my_row = r0 + rg + cg * RG;
        if (cg < RPT && my_row < p.rows)
            p.row_d[my_row * p.rd_row + ((shift + c0) / G) * p.rd_blk] = __fdiv_rn(mine, FMAX);
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            const float hi = __shfl_sync(0xffffffffu, scale.hi, (lane & 16) | i);
            float lo = 0.0f;
            if constexpr (IsPacked<Tile>::value) lo = __shfl_sync(0xffffffffu, scale.lo, (lane & 16) | i);
            const int r = r0 + rg + i * RG;
            if (r < p.rows && n > 0) {
                float f[8];
                t.row(i, f);
                uint2 q;
                if constexpr (IsPacked<Tile>::value) q = code8x<E5M2>(f, hi, lo);
                else q = code8<E5M2>(f, hi);
                store8(p.row8 + static_cast<long long>(r) * p.ld_row8 + shift + col, q, n, p.vec_row8);
            }
        }
    }
    if (COL) {
        __syncthreads();
        float* s_scale = s_col + (T / 32) * G;               // of the 128 columns (packed tiles: hi, then lo)
        if (threadIdx.x < G) {
            float a = s_col[threadIdx.x];
#pragma unroll
            for (int w = 1; w < T / 32; ++w) a = fmaxf(a, s_col[w * G + threadIdx.x]);
            a = fmaxf(a, kFloorAmax);
            if constexpr (IsPacked<Tile>::value) {
                const Scale2 sc = scale2(FMAX, a);
                s_scale[threadIdx.x] = sc.hi;
                s_scale[G + threadIdx.x] = sc.lo;
            } else {
                s_scale[threadIdx.x] = __fdiv_rn(FMAX, a);
            }
            if (c0 + static_cast<int>(threadIdx.x) < p.cols)
                p.col_d[(r0 / G) * p.cd_blk + static_cast<long long>(shift + c0 + threadIdx.x) * p.cd_col] = __fdiv_rn(a, FMAX);
        }
        __syncthreads();
        float s[8];
        const float4 lo = *reinterpret_cast<const float4*>(s_scale + cg * 8), hi = *reinterpret_cast<const float4*>(s_scale + cg * 8 + 4);
        s[0] = lo.x; s[1] = lo.y; s[2] = lo.z; s[3] = lo.w; s[4] = hi.x; s[5] = hi.y; s[6] = hi.z; s[7] = hi.w;
        float s_lo[8];
        if constexpr (IsPacked<Tile>::value) {
#pragma unroll
            for (int e = 0; e < 8; ++e) s_lo[e] = s_scale[G + cg * 8 + e];
        }
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            const int r = r0 + rg + i * RG;
            if (r < p.rows && n > 0) {
                float f[8];
                t.row(i, f);
                if constexpr (IsPacked<Tile>::value) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[e] = fmaf(f[e], s_lo[e], f[e] * s[e]);
                    store8(p.col8 + static_cast<long long>(r) * p.ld_col8 + shift + col, code8<E5M2>(f, 1.0f), n, p.vec_col8);
                } else {
                    store8(p.col8 + static_cast<long long>(r) * p.ld_col8 + shift + col, code8c<E5M2>(f, s), n, p.vec_col8);
                }
            }
        }
    }
}

// Tile of (T / 16) * RPT rows x 128 columns. With column groups the tile has 128 rows. The second launch bound holds the
// registers down to where enough blocks share an SM to hide the loads: SwiGLU rows, 2039 x 14336: 38.6 us at 64 registers (four
// blocks of 256 threads), 37.1 at 48, 35.0 at 40 (six); one row a thread instead of two 42. As it is 35.4 us, since gates of any
// size are right.
template <int SRC, int T, int RPT, bool ROW, bool COL, bool E5M2>
__global__ void __launch_bounds__(T, !COL ? (SRC == SRC_SWIGLU ? 1536 : 1024) / T : SRC == SRC_PLAIN ? 3 : 2) k_quant_block128(const QuantParams p) {
    constexpr int RG = T / 16;
    __shared__ __align__(16) float s_col[COL ? (T / 32 + 2) * G : 4];
    const int cb = blockIdx.x % p.col_blocks, rb = blockIdx.x / p.col_blocks;
    const int c0 = cb * G, r0 = rb * (RG * RPT);
    const int cg = threadIdx.x & 15, rg = threadIdx.x >> 4;
    const int col = c0 + cg * 8;
    const int n = min(8, p.cols - col);

    pdl_wait();
    uint4 b[SRC == SRC_SWIGLU ? RPT : 1];
    PackedTile<RPT> a;
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
        const int r = r0 + rg + i * RG;
        a.v[i] = make_uint4(0u, 0u, 0u, 0u);
        if (SRC == SRC_SWIGLU) b[i] = a.v[i];
        if (r < p.rows && n > 0) {
            a.v[i] = load8(p.x + r * p.ld_x + col, n, p.vec_in);
            if (SRC == SRC_SWIGLU) b[i] = load8(p.up + r * p.ld_x + col, n, p.vec_in);
        }
    }
    if constexpr (SRC == SRC_PLAIN) {
        emit_tile<T, RPT, ROW, COL, E5M2>(p, a, r0, c0, 0, s_col);
    } else {
        FloatTile<RPT> f;
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            float g[8], u[8];
            unpack8(a.v[i], g);
            unpack8(b[i], u);
#pragma unroll
            for (int e = 0; e < 8; ++e) f.v[i][e] = swiglu(g[e], u[e]);
        }
        emit_tile<T, RPT, ROW, COL, E5M2>(p, f, r0, c0, 0, s_col);
    }
}

// Gradient of silu(gate) * up, the two halves of one [rows, 2 cols] gradient. With e = exp(-g), s = sig(g) = 1 / (1 + e) and
// 1 - s = e s (no cancellation where s is near one):
//   d gate = dh up s (1 + g e s),  d up = dh g s
// A tile's three inputs wait in shared memory, each thread's own 16-byte pieces (asynchronous copies, no barrier): held in
// registers they leave room for one block per SM, whose loads and arithmetic then do not overlap. d up is kept in the place of
// gate and up until d gate has left, so the exponential is taken once. 4096 x 14336, both groupings: 237 us with the inputs in
// registers, 120 to 132 us now (by the box).
constexpr int kGradT = 512, kGradRPT = G / (kGradT / 16);
constexpr int kGradSmem = 3 * kGradRPT * kGradT * 16;
template <bool ROW, bool COL, bool E5M2>
__global__ void __launch_bounds__(kGradT, 2) k_swiglu_grad_block128(const QuantParams p) {
    constexpr int RG = kGradT / 16;
    extern __shared__ __align__(16) uint4 s_in[];              // [gate, up, dh][row][thread]
    __shared__ __align__(16) float s_col[2][COL ? (kGradT / 32 + 1) * G : 4];      // a copy per half: no barrier between them
    const int cb = blockIdx.x % p.col_blocks, rb = blockIdx.x / p.col_blocks;
    const int c0 = cb * G, r0 = rb * G;
    const int cg = threadIdx.x & 15, rg = threadIdx.x >> 4;
    const int col = c0 + cg * 8;                               // cols is a multiple of 128: every vector is whole
    pdl_wait();
#pragma unroll
    for (int i = 0; i < kGradRPT; ++i) {
        const int r = r0 + rg + i * RG;
        const uint16_t* src[3] = {p.x + r * p.ld_x + col, p.up + r * p.ld_x + col, p.dh + r * p.ld_dh + col};
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            uint4* d = s_in + (k * kGradRPT + i) * kGradT + threadIdx.x;
            if (r < p.rows && p.vec_in) {
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(d))), "l"(src[k]) : "memory");
            } else {
                *d = r < p.rows ? load8(src[k], 8, false) : make_uint4(0u, 0u, 0u, 0u);
            }
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    FloatTile<kGradRPT> f;
#pragma unroll
    for (int i = 0; i < kGradRPT; ++i) {
        uint4* own[3] = {s_in + i * kGradT + threadIdx.x, s_in + (kGradRPT + i) * kGradT + threadIdx.x,
                         s_in + (2 * kGradRPT + i) * kGradT + threadIdx.x};
        float g[8], u[8], d[8];
        unpack8(*own[0], g);
        unpack8(*own[1], u);
        unpack8(*own[2], d);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float ex = fminf(expf(-g[e]), FLT_MAX);      // finite: far below zero s is 0 and e s is too, not inf * 0
            const float r0 = rcp(1.0f + ex), sg = fmaf(fmaf(-(1.0f + ex), r0, 1.0f), r0, r0);
            const float ds = d[e] * sg;
            f.v[i][e] = ds * u[e] * fmaf(g[e], ex * sg, 1.0f);
            d[e] = ds * g[e];
        }
        *reinterpret_cast<float4*>(own[0]) = make_float4(d[0], d[1], d[2], d[3]);
        *reinterpret_cast<float4*>(own[1]) = make_float4(d[4], d[5], d[6], d[7]);
    }
    emit_tile<kGradT, kGradRPT, ROW, COL, E5M2>(p, f, r0, c0, 0, s_col[0]);
#pragma unroll
    for (int i = 0; i < kGradRPT; ++i) {
        const float4 lo = *reinterpret_cast<const float4*>(s_in + i * kGradT + threadIdx.x);
        const float4 hi = *reinterpret_cast<const float4*>(s_in + (kGradRPT + i) * kGradT + threadIdx.x);
        f.v[i][0] = lo.x; f.v[i][1] = lo.y; f.v[i][2] = lo.z; f.v[i][3] = lo.w;
        f.v[i][4] = hi.x; f.v[i][5] = hi.y; f.v[i][6] = hi.z; f.v[i][7] = hi.w;
    }
    emit_tile<kGradT, kGradRPT, ROW, COL, E5M2>(p, f, r0, c0, p.cols, s_col[1]);
}

// Weights: one scale per 128x128 block of every [rows, cols] matrix of a stack (blocks restart in each matrix).
constexpr int kWT = 512;
__global__ void __launch_bounds__(kWT) k_quant_block128x128(const uint16_t* __restrict__ w, long long ld_w, long long w_stride, int rows,
                                                            int cols, int row_blocks, int col_blocks, uint8_t* __restrict__ out,
                                                            long long ld_out, long long out_stride, float* __restrict__ descale,
                                                            long long d_row, long long d_stride, int vec_in, int vec_out) {
    constexpr int RG = kWT / 16, RPT = G / RG;
    __shared__ float s_part[kWT / 32];
    const int cb = blockIdx.x % col_blocks;
    const int t = blockIdx.x / col_blocks;
    const int rb = t % row_blocks, m = t / row_blocks;
    const int cg = threadIdx.x & 15, rg = threadIdx.x >> 4;
    const int col = cb * G + cg * 8;
    const int n = min(8, cols - col);
    const uint16_t* src = w + m * w_stride;
    uint4 v[RPT];
    float a = 0.0f;
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
        const int r = rb * G + rg + i * RG;
        v[i] = make_uint4(0u, 0u, 0u, 0u);
        if (r < rows && n > 0) v[i] = load8(src + r * ld_w + col, n, vec_in);
    }
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
        float f[8];
        unpack8(v[i], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) a = fmaxf(a, fabsf(f[e]));
    }
    a = warp_max(a);
    if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = a;
    __syncthreads();
    a = s_part[0];
#pragma unroll
    for (int i = 1; i < kWT / 32; ++i) a = fmaxf(a, s_part[i]);
    a = fmaxf(a, kFloorAmax);
    const Scale2 s = scale2(448.0f, a);
    if (threadIdx.x == 0) descale[m * d_stride + rb * d_row + cb] = __fdiv_rn(a, 448.0f);
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
        const int r = rb * G + rg + i * RG;
        if (r < rows && n > 0) {
            float f[8];
            unpack8(v[i], f);
            store8(out + m * out_stride + r * ld_out + col, code8x<false>(f, s.hi, s.lo), n, vec_out);
        }
    }
}

// ------------------------------------------------------------------ host side
bool aligned(const void* p, uintptr_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }
long long cdiv(long long a, long long b) { return (a + b - 1) / b; }

long long tiles(const QuantParams& p, int rows_per_tile) { return cdiv(p.rows, rows_per_tile) * p.col_blocks; }
bool fits(long long blocks) {
    if (blocks <= 0x7fffffffll) return true;
    set_error("block-128 quantiser: matrix too large for one launch");
    return false;
}

template <int SRC, int T, int RPT, bool ROW, bool COL>
int launch_fmt(const QuantParams& p, int e5m2, cudaStream_t st) {
    const long long blocks = tiles(p, (T / 16) * RPT);
    if (!fits(blocks)) return CF_ERR_LIMIT;
    const dim3 grid(static_cast<unsigned>(blocks));
    if constexpr (SRC == SRC_SWIGLU) {
        CF_CUDA(launch_pdl(k_quant_block128<SRC, T, RPT, ROW, COL, false>, grid, dim3(T), 0, st, p));       // E4M3 only
    } else {
        CF_CUDA(e5m2 ? launch_pdl(k_quant_block128<SRC, T, RPT, ROW, COL, true>, grid, dim3(T), 0, st, p)
                     : launch_pdl(k_quant_block128<SRC, T, RPT, ROW, COL, false>, grid, dim3(T), 0, st, p));
    }
    CF_LAUNCH_CHECK("quant_block128");
    return CF_OK;
}

template <bool ROW, bool COL, bool E5M2>
int launch_grad(const QuantParams& p, cudaStream_t st) {
    const long long blocks = tiles(p, G);
    if (!fits(blocks)) return CF_ERR_LIMIT;
    static std::atomic<int> ready[64];                  // the attribute is set once per device (any thread may do it)
    int dev = 0;
    CF_CUDA(cudaGetDevice(&dev));
    if (!ready[dev & 63].load(std::memory_order_acquire)) {
        CF_CUDA(cudaFuncSetAttribute(k_swiglu_grad_block128<ROW, COL, E5M2>, cudaFuncAttributeMaxDynamicSharedMemorySize, kGradSmem));
        ready[dev & 63].store(1, std::memory_order_release);
    }
    CF_CUDA(launch_pdl(k_swiglu_grad_block128<ROW, COL, E5M2>, dim3(static_cast<unsigned>(blocks)), dim3(kGradT), kGradSmem, st, p));
    CF_LAUNCH_CHECK("swiglu_grad_block128");
    return CF_OK;
}

template <int SRC>
int launch_quant(const char* fn, QuantParams p, int e5m2, int halves, cudaStream_t st) {
    CF_REQUIRE(p.rows >= 0 && p.cols >= 0, "%s: negative shape", fn);
    if (p.rows == 0 || p.cols == 0) return CF_OK;
    if (p.rows > 0x7fff0000 || p.cols > 0x3fff0000) { set_error("%s: more than 2^31 rows or 2^30 columns", fn); return CF_ERR_LIMIT; }
    const bool row = p.row8 != nullptr, col = p.col8 != nullptr;
    CF_REQUIRE(row || col, "%s: no output", fn);
    CF_REQUIRE(row == (p.row_d != nullptr) && col == (p.col_d != nullptr), "%s: codes and descales go together", fn);
    CF_REQUIRE(p.x && (SRC == SRC_PLAIN || p.up) && (SRC != SRC_SWIGLU_GRAD || p.dh), "%s: null input", fn);
    CF_REQUIRE(p.ld_x >= p.cols && (SRC != SRC_SWIGLU_GRAD || p.ld_dh >= p.cols), "%s: input pitch smaller than a row", fn);
    CF_REQUIRE((!row || p.ld_row8 >= static_cast<long long>(halves) * p.cols) && (!col || p.ld_col8 >= static_cast<long long>(halves) * p.cols),
               "%s: output pitch smaller than a row", fn);
    CF_REQUIRE(halves == 1 || p.cols % G == 0, "%s: the two halves need cols to be a multiple of 128", fn);
    CF_REQUIRE(aligned(p.x, 2) && aligned(p.up, 2) && aligned(p.dh, 2) && aligned(p.row_d, 4) && aligned(p.col_d, 4),
               "%s: misaligned pointer", fn);
    const int rc = require_sm100();
    if (rc != CF_OK) return rc;
    p.col_blocks = static_cast<int>(cdiv(p.cols, G));
    p.vec_in = aligned(p.x, 16) && aligned(p.up, 16) && aligned(p.dh, 16) && p.ld_x % 8 == 0 && (SRC != SRC_SWIGLU_GRAD || p.ld_dh % 8 == 0);
    p.vec_row8 = row && aligned(p.row8, 8) && p.ld_row8 % 8 == 0;
    p.vec_col8 = col && aligned(p.col8, 8) && p.ld_col8 % 8 == 0;
    if constexpr (SRC == SRC_SWIGLU_GRAD) {
        if (col && row) return e5m2 ? launch_grad<true, true, true>(p, st) : launch_grad<true, true, false>(p, st);
        if (col) return e5m2 ? launch_grad<false, true, true>(p, st) : launch_grad<false, true, false>(p, st);
        return e5m2 ? launch_grad<true, false, true>(p, st) : launch_grad<true, false, false>(p, st);
    } else {
        if (col && row) return launch_fmt<SRC, 512, 4, true, true>(p, e5m2, st);
        if (col) return launch_fmt<SRC, 512, 4, false, true>(p, e5m2, st);
        // Rows alone: tiles of 64 rows (SwiGLU: 32) amortise a thread's divisions over its rows; with fewer than two such tiles per SM
        // tiles of 8 rows spread the work over more of them (one row of 14336 columns then takes 112 small blocks).
        constexpr int kRows = SRC == SRC_PLAIN ? 4 : 2;
        if (tiles(p, 16 * kRows) >= 2ll * sm_count()) return launch_fmt<SRC, 256, kRows, true, false>(p, e5m2, st);
        return launch_fmt<SRC, 128, 1, true, false>(p, e5m2, st);
    }
}

}  // namespace
}  // namespace cf

using namespace cf;

extern "C" {

int cf_fp8_quantize_block128(const void* d_x, int ld_x, int rows, int cols, int is_e5m2, void* d_row8_or_null, int ld_row8,
                             float* d_row_descale, long long row_descale_ld_row, long long row_descale_ld_block, void* d_col8_or_null,
                             int ld_col8, float* d_col_descale, long long col_descale_ld_block, long long col_descale_ld_col, void* stream) {
    QuantParams p = {};
    p.x = static_cast<const uint16_t*>(d_x); p.ld_x = ld_x; p.rows = rows; p.cols = cols;
    p.row8 = static_cast<uint8_t*>(d_row8_or_null); p.ld_row8 = ld_row8;
    p.row_d = d_row_descale; p.rd_row = row_descale_ld_row; p.rd_blk = row_descale_ld_block;
    p.col8 = static_cast<uint8_t*>(d_col8_or_null); p.ld_col8 = ld_col8;
    p.col_d = d_col_descale; p.cd_blk = col_descale_ld_block; p.cd_col = col_descale_ld_col;
    return launch_quant<SRC_PLAIN>("cf_fp8_quantize_block128", p, is_e5m2, 1, as_stream(stream));
}

int cf_swiglu_quantize_block128(const void* d_gate, const void* d_up, int ld_in, int rows, int cols, void* d_row8_or_null, int ld_row8,
                                float* d_row_descale, long long row_descale_ld_row, long long row_descale_ld_block,
                                void* d_col8_or_null, int ld_col8, float* d_col_descale, long long col_descale_ld_block,
                                long long col_descale_ld_col, void* stream) {
    QuantParams p = {};
    p.x = static_cast<const uint16_t*>(d_gate); p.up = static_cast<const uint16_t*>(d_up);
    p.ld_x = ld_in; p.rows = rows; p.cols = cols;
    p.row8 = static_cast<uint8_t*>(d_row8_or_null); p.ld_row8 = ld_row8;
    p.row_d = d_row_descale; p.rd_row = row_descale_ld_row; p.rd_blk = row_descale_ld_block;
    p.col8 = static_cast<uint8_t*>(d_col8_or_null); p.ld_col8 = ld_col8;
    p.col_d = d_col_descale; p.cd_blk = col_descale_ld_block; p.cd_col = col_descale_ld_col;
    return launch_quant<SRC_SWIGLU>("cf_swiglu_quantize_block128", p, 0, 1, as_stream(stream));
}

int cf_swiglu_backward_quantize_block128(const void* d_gate, const void* d_up, int ld_in, const void* d_dh, int ld_dh, int rows, int cols,
                                         int is_e5m2, void* d_row8_or_null, int ld_row8, float* d_row_descale,
                                         long long row_descale_ld_row, long long row_descale_ld_block, void* d_col8_or_null,
                                         int ld_col8, float* d_col_descale, long long col_descale_ld_block, long long col_descale_ld_col,
                                         void* stream) {
    QuantParams p = {};
    p.x = static_cast<const uint16_t*>(d_gate); p.up = static_cast<const uint16_t*>(d_up); p.dh = static_cast<const uint16_t*>(d_dh);
    p.ld_x = ld_in; p.ld_dh = ld_dh; p.rows = rows; p.cols = cols;
    p.row8 = static_cast<uint8_t*>(d_row8_or_null); p.ld_row8 = ld_row8;
    p.row_d = d_row_descale; p.rd_row = row_descale_ld_row; p.rd_blk = row_descale_ld_block;
    p.col8 = static_cast<uint8_t*>(d_col8_or_null); p.ld_col8 = ld_col8;
    p.col_d = d_col_descale; p.cd_blk = col_descale_ld_block; p.cd_col = col_descale_ld_col;
    return launch_quant<SRC_SWIGLU_GRAD>("cf_swiglu_backward_quantize_block128", p, is_e5m2, 2, as_stream(stream));
}

int cf_fp8_quantize_block128x128(const void* d_w, int ld_w, long long w_stride, int num_weights, int rows, int cols, void* d_out8,
                                 int ld_out, long long out_stride, float* d_descale, long long descale_ld_row, long long descale_stride,
                                 void* stream) {
    const char* fn = "cf_fp8_quantize_block128x128";
    CF_REQUIRE(num_weights >= 0 && rows >= 0 && cols >= 0, "%s: negative shape", fn);
    if (num_weights == 0 || rows == 0 || cols == 0) return CF_OK;
    CF_REQUIRE(d_w && d_out8 && d_descale, "%s: null pointer", fn);
    CF_REQUIRE(ld_w >= cols && ld_out >= cols && descale_ld_row >= cdiv(cols, G), "%s: pitch smaller than a row", fn);
    CF_REQUIRE(num_weights == 1 || (w_stride >= static_cast<long long>(rows - 1) * ld_w + cols &&
                                    out_stride >= static_cast<long long>(rows - 1) * ld_out + cols &&
                                    descale_stride >= (cdiv(rows, G) - 1) * descale_ld_row + cdiv(cols, G)),
               "%s: matrices of the stack overlap", fn);
    CF_REQUIRE(aligned(d_w, 2) && aligned(d_descale, 4), "%s: misaligned pointer", fn);
    const int rc = require_sm100();
    if (rc != CF_OK) return rc;
    const int rb = static_cast<int>(cdiv(rows, G)), cb = static_cast<int>(cdiv(cols, G));
    const long long blocks = static_cast<long long>(num_weights) * rb * cb;
    if (blocks > 0x7fffffffll) { set_error("%s: too many blocks for one launch", fn); return CF_ERR_LIMIT; }
    const int vec_in = aligned(d_w, 16) && ld_w % 8 == 0 && (num_weights == 1 || w_stride % 8 == 0);
    const int vec_out = aligned(d_out8, 8) && ld_out % 8 == 0 && (num_weights == 1 || out_stride % 8 == 0);
    k_quant_block128x128<<<static_cast<unsigned>(blocks), kWT, 0, as_stream(stream)>>>(
        static_cast<const uint16_t*>(d_w), ld_w, w_stride, rows, cols, rb, cb, static_cast<uint8_t*>(d_out8), ld_out, out_stride,
        d_descale, descale_ld_row, descale_stride, vec_in, vec_out);
    CF_LAUNCH_CHECK("quant_block128x128");
    return CF_OK;
}

}  // extern "C"
