// Residual addition + RMS norm with block-scaled FP8 output, and the gradient of the pair.
//
//   forward   h = bf16(x + residual);  rms = sqrt(mean(h^2) + eps);  y = (h / rms) * scale
//             per 128 values of y: a = max(max|y|, 1e-12), descale = a / 448, code = e4m3(y * 448 / a)
//   backward  u = dy * scale;  dx = (u - h * sum(u h) / (H rms^2)) / rms + dh;  dscale = sum over rows of dy * h / rms
//
// h is rounded to bf16 before the norm reads it: it is the residual stream the next layers and the backward pass see. y is
// NOT rounded to bf16 on its way to the codes (one rounding, descales from fp32); the optional bf16 copy of y is. The codes do
// not depend on rms: with t = h * scale (exact in fp32, 16 bits) and m = max|t| over the group, y * 448 / a = t * 448 / m. The
// quotient is taken correctly rounded, exact where it is representable: it lands exactly between two codes about once in a
// thousand values, and a rounded factor would send such a value to either side.
// Sums, rms and descales are fp32; a sum of squares beyond fp32 is taken again over scaled values. In a row with an infinity rms is
// infinite and y is 0, NaN at the infinity itself; a NaN makes its whole row NaN.
//
// Both are streams: forward 2+2 B in, 2+1 B out per element (7), backward 2+2+2 in, 2 out (8). A row lives in the registers
// of one block between its reduction and its second use, 16 neighbouring threads hold one group of 128, and one block
// barrier per row joins the row sum (two copies of the partial sums alternate, so the next row needs no second barrier).
// The gain's gradient is summed per block over the block's rows in registers, written as one partial row per block and
// added up in block order by a second launch: no atomics, so the result does not depend on timing. The launches may be scheduled
// while the kernel before them drains (they wait for it before they touch memory): the gradient of 8192 x 4096 and its sum take
// 50 us instead of 53 (52 on another box).
#include <type_traits>

#include "cf_common.cuh"
#include "cf_internal.cuh"

namespace cf {
namespace {

constexpr int kMaxH = 16384;
constexpr int kBwdBlocks = 148;             // per block that an SM holds: fixed, so that the order of the sums does not follow the device

__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
    f[0] = __uint_as_float(v.x << 16); f[1] = __uint_as_float(v.x & 0xffff0000u);
    f[2] = __uint_as_float(v.y << 16); f[3] = __uint_as_float(v.y & 0xffff0000u);
    f[4] = __uint_as_float(v.z << 16); f[5] = __uint_as_float(v.z & 0xffff0000u);
    f[6] = __uint_as_float(v.w << 16); f[7] = __uint_as_float(v.w & 0xffff0000u);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
    return make_uint4(pack2(f[0], f[1]), pack2(f[2], f[3]), pack2(f[4], f[5]), pack2(f[6], f[7]));
}
// VEC: whole 16-byte vectors (H % 8 == 0 and aligned rows); otherwise element by element, n of 8 valid.
template <bool VEC>
__device__ __forceinline__ uint4 load8(const uint16_t* p, int n) {
    if (VEC) return *reinterpret_cast<const uint4*>(p);
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e < n) w[e >> 1] |= static_cast<uint32_t>(p[e]) << (16 * (e & 1));
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <bool VEC>
__device__ __forceinline__ void store8(uint16_t* p, const uint4& v, int n) {
    if (VEC) { *reinterpret_cast<uint4*>(p) = v; return; }
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e < n) p[e] = static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1)));
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
}
// Sum over the block, the same value in every thread; `slot` is the copy of the partial sums this row uses.
__device__ __forceinline__ float block_sum(float v, float* slot) {
    v = warp_sum(v);
    if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
    __syncthreads();
    const int nw = blockDim.x >> 5;
    float t = 0.0f;
    for (int w = 0; w < nw; ++w) t += slot[w];
    return t;
}

struct NormParams {
    const uint16_t* x;
    const uint16_t* res;
    const uint16_t* gain;
    uint16_t* h;
    uint16_t* normed;
    float* rms;
    uint8_t* out8;
    long long ld_out8;
    float* descale;
    long long d_row, d_blk;
    int rows, H;
    float eps;
    int vec8;
};

// 448 / m in two parts, 8 significant bits and the rest: t * hi is exact, fma(t, lo, t * hi) the rounded quotient.
struct Quotient { float hi, lo; };
__device__ __forceinline__ Quotient quotient(float m) {
    const float quot = __fdiv_rn(448.0f, m);
    const float hi = __uint_as_float(__float_as_uint(quot) & 0xffff0000u);
    const float rest = fmaf(fmaf(-quot, m, 448.0f), quot * (1.0f / 448.0f), quot - hi);
    return {hi, isfinite(rest) ? rest : 0.0f};          // a group with an infinity: the quotient is 0
}

// A row whose sum of squares is beyond fp32, by all threads of its block. Values above 1.8e19 alone do that: the sum is taken again
// over h * 2^-72 (below 2^126 for the longest row of the largest numbers; what loses bits in the scaling is below 2^-110 of the rms),
// and y = (h 2^-72) / (rms 2^-72) * scale. With an infinity or a NaN in the row that sum is not finite either: y = h / rms * scale
// is then taken before the groups' maxima (a factor of 1 / rms behind them would be inf * 0 in every group).
// The row is read again from where h stands, the sum's barrier has made it visible; a call of its own, since lines inside the
// kernel cost every row (16384 x 4096: 84 us instead of 80).
__device__ __noinline__ void unbounded_row(const NormParams& p, long long row) {
    constexpr float kDown = 0x1p-72f, kUp = 0x1p72f;
    __shared__ float s_again[32];
    const uint16_t* src = (p.h ? p.h : p.x) + row * p.H;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    float acc = 0.0f;
    for (int c = threadIdx.x; c < p.H; c += blockDim.x) {
        const float f = bf16_bits_to_f32(src[c]) * kDown;
        acc = fmaf(f, f, acc);
    }
    float rms = sqrtf(__fdiv_rn(block_sum(acc, s_again), static_cast<float>(p.H)) + p.eps * kDown * kDown);
    if (threadIdx.x == 0 && p.rms) p.rms[row] = rms * kUp;
    float inv = __fdiv_rn(1.0f, rms), factor = kDown;        // t = h * factor * scale, y = t * inv
    if (!isfinite(rms)) {
        factor = inv;
        rms = inv = 1.0f;
    }
    for (int group = warp; group * 128 < p.H; group += warps) {      // one warp: 128 values, four a lane
        float t[4], m = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int c = group * 128 + 32 * e + lane;
            t[e] = c < p.H ? bf16_bits_to_f32(src[c]) * factor * bf16_bits_to_f32(p.gain[c]) : 0.0f;
            m = fmaxf(m, fabsf(t[e]));
        }
        m = fmaxf(warp_max(m), 1e-12f * rms);
        const Quotient q = quotient(m);
        if (p.out8 && lane == 0) p.descale[row * p.d_row + group * p.d_blk] = __fdiv_rn(m * inv, 448.0f);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int c = group * 128 + 32 * e + lane;
            if (c < p.H) {
                if (p.normed) p.normed[row * p.H + c] = static_cast<uint16_t>(pack2(t[e] * inv, 0.0f));
                if (p.out8) p.out8[row * p.ld_out8 + c] = cvt_fp8<false>(fmaf(t[e], q.lo, t[e] * q.hi));
            }
        }
    }
}

// x, res and h may be the same memory (every thread reads its own elements before it writes them, and a row belongs to one
// block): no __restrict__. A row's loads of x and of the residual are all issued before either is used: 16384 x 4096 takes
// 78 to 80 us (0.90 to 0.92 of the measured copy rate), 89 with the residual's loads behind the use of x's.
template <int NV, bool VEC>
__global__ void __launch_bounds__(1024) k_add_rmsnorm(const __grid_constant__ NormParams p) {
    __shared__ float s_sum[2][32];
    const int nv = (p.H + 7) / 8;
    pdl_wait();
    int par = 0;
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x, par ^= 1) {
        const long long base = row * p.H;
        uint4 v[NV], res[NV];
        float acc = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int vi = threadIdx.x + blockDim.x * i;
            v[i] = res[i] = make_uint4(0u, 0u, 0u, 0u);
            if (vi < nv) {
                v[i] = load8<VEC>(p.x + base + vi * 8, p.H - vi * 8);
                if (p.res) res[i] = load8<VEC>(p.res + base + vi * 8, p.H - vi * 8);
            }
        }
        if (p.res) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                float a[8], b[8];
                unpack8(v[i], a);
                unpack8(res[i], b);
#pragma unroll
                for (int e = 0; e < 8; ++e) a[e] += b[e];
                v[i] = pack8(a);
            }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float f[8];
            unpack8(v[i], f);
#pragma unroll
            for (int e = 0; e < 8; ++e) acc = fmaf(f[e], f[e], acc);
            const int vi = threadIdx.x + blockDim.x * i;
            if (p.h && vi < nv) store8<VEC>(p.h + base + vi * 8, v[i], p.H - vi * 8);
        }
        const float total = block_sum(acc, s_sum[par]);
        const float rms = sqrtf(__fdiv_rn(total, static_cast<float>(p.H)) + p.eps);
        if (!isfinite(rms)) {                           // the same in every thread
            unbounded_row(p, row);
            continue;
        }
        if (threadIdx.x == 0 && p.rms) p.rms[row] = rms;
        const float inv = __fdiv_rn(1.0f, rms);
        float amax[NV];                                 // of t over the group of 128 that this half-warp holds in vector i
        float t[NV][8];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int vi = threadIdx.x + blockDim.x * i;
            float g[8];
            unpack8(v[i], t[i]);
            unpack8(vi < nv ? load8<VEC>(p.gain + vi * 8, p.H - vi * 8) : make_uint4(0u, 0u, 0u, 0u), g);
            amax[i] = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                t[i][e] *= g[e];
                amax[i] = fmaxf(amax[i], fabsf(t[i][e]));
            }
            if (p.normed && vi < nv) {
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = t[i][e] * inv;
                store8<VEC>(p.normed + base + vi * 8, pack8(y), p.H - vi * 8);
            }
        }
        if (p.out8) {                                   // kernel-uniform
#pragma unroll
            for (int i = 0; i < NV; ++i) {
#pragma unroll
                for (int off = 8; off > 0; off >>= 1) amax[i] = fmaxf(amax[i], __shfl_xor_sync(0xffffffffu, amax[i], off));
            }
            // lane i of a half-warp divides for group i, the quotients are handed round
            const int lane = threadIdx.x & 31, cg = lane & 15;
            float mine = amax[0];
#pragma unroll
            for (int i = 1; i < NV; ++i)
                if (cg == i) mine = amax[i];
            mine = fmaxf(mine, 1e-12f * rms);           // the floor of max|y|
            const Quotient s = quotient(mine);
            const int my_group = (threadIdx.x + blockDim.x * cg) / 16;
            if (cg < NV && my_group * 16 < nv) p.descale[row * p.d_row + my_group * p.d_blk] = __fdiv_rn(mine * inv, 448.0f);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int vi = threadIdx.x + blockDim.x * i;
                const float hi = __shfl_sync(0xffffffffu, s.hi, (lane & 16) | i), lo = __shfl_sync(0xffffffffu, s.lo, (lane & 16) | i);
                if (vi < nv) {
                    float q[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) q[e] = fmaf(t[i][e], lo, t[i][e] * hi);
                    const uint32_t q0 = cvt_fp8x4<false>(q[0], q[1], q[2], q[3]);
                    const uint32_t q1 = cvt_fp8x4<false>(q[4], q[5], q[6], q[7]);
                    uint8_t* o = p.out8 + row * p.ld_out8 + vi * 8;
                    if (VEC && p.vec8) {
                        *reinterpret_cast<uint2*>(o) = make_uint2(q0, q1);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (vi * 8 + e < p.H) o[e] = static_cast<uint8_t>((e < 4 ? q0 >> (8 * e) : q1 >> (8 * (e - 4))) & 0xffu);
                    }
                }
            }
        }
    }
}

struct NormGradParams {
    const uint16_t* dy;
    const uint16_t* h;
    const uint16_t* gain;
    const float* rms;
    const uint16_t* dh;
    uint16_t* dx;
    float* partial;           // [gridDim.x, H] or null
    int rows, H;
};

// dx may be the same memory as dy or dh. The next row's loads are issued before this row's barrier, except with four vectors a
// thread, which leave no registers for it. Two resident blocks with one vector, one block (128 registers a thread) otherwise.
template <int NV, bool VEC>
__global__ void __launch_bounds__(512, NV == 1 ? 2 : 1) k_add_rmsnorm_grad(const NormGradParams p) {
    constexpr bool PREFETCH = NV <= 2;
    __shared__ float s_sum[2][32];
    const int nv = (p.H + 7) / 8;
    pdl_wait();
    float dg[NV][8];
    uint4 gain[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int vi = threadIdx.x + blockDim.x * i;
        gain[i] = vi < nv ? load8<VEC>(p.gain + vi * 8, p.H - vi * 8) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int e = 0; e < 8; ++e) dg[i][e] = 0.0f;
    }
    struct Row { uint4 dy[NV], h[NV], dh[NV]; float rms; };
    auto load = [&](Row& r, long long row) {
        const long long base = row * p.H;
        r.rms = p.rms[row];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int vi = threadIdx.x + blockDim.x * i;
            r.dy[i] = r.h[i] = r.dh[i] = make_uint4(0u, 0u, 0u, 0u);
            if (vi < nv) {
                r.dy[i] = load8<VEC>(p.dy + base + vi * 8, p.H - vi * 8);
                r.h[i] = load8<VEC>(p.h + base + vi * 8, p.H - vi * 8);
                if (p.dh) r.dh[i] = load8<VEC>(p.dh + base + vi * 8, p.H - vi * 8);
            }
        }
    };
    int par = 0;
    Row r, next;
    if (PREFETCH && blockIdx.x < p.rows) load(r, blockIdx.x);
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x, par ^= 1) {
        if (!PREFETCH) load(r, row);
        else if (row + gridDim.x < p.rows) load(next, row + gridDim.x);
        const float inv = __fdiv_rn(1.0f, r.rms);
        float acc = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float a[8], b[8], g[8];
            unpack8(r.dy[i], a);
            unpack8(r.h[i], b);
            unpack8(gain[i], g);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                acc = fmaf(a[e] * g[e], b[e] * inv, acc);
                dg[i][e] = fmaf(a[e], b[e] * inv, dg[i][e]);
            }
        }
        const float mean = __fdiv_rn(block_sum(acc, s_sum[par]), static_cast<float>(p.H));
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int vi = threadIdx.x + blockDim.x * i;
            float a[8], b[8], g[8], d[8];
            unpack8(r.dy[i], a);
            unpack8(r.h[i], b);
            unpack8(gain[i], g);
            unpack8(r.dh[i], d);
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e] = fmaf(fmaf(-b[e] * inv, mean, a[e] * g[e]), inv, d[e]);
            if (vi < nv) store8<VEC>(p.dx + row * p.H + vi * 8, pack8(d), p.H - vi * 8);
        }
        if (PREFETCH) r = next;
    }
    if (p.partial) {
        float* o = p.partial + static_cast<long long>(blockIdx.x) * p.H;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int vi = threadIdx.x + blockDim.x * i;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (vi * 8 + e < p.H) o[vi * 8 + e] = dg[i][e];
        }
    }
}

// out[c] (+)= sum over the partial rows, in row order within each of the 32 warps of a block, then over the warps.
__global__ void __launch_bounds__(1024) k_sum_partials(const float* partial, int n, int H, float* out, int accumulate) {
    __shared__ float s[32][33];
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + lane;
    float t = 0.0f;
    if (c < H)
#pragma unroll 8
        for (int r = warp; r < n; r += 32) t += partial[static_cast<long long>(r) * H + c];
    s[warp][lane] = t;
    __syncthreads();
    if (warp == 0 && c < H) {
        float v = s[0][lane];
#pragma unroll
        for (int w = 1; w < 32; ++w) v += s[w][lane];
        out[c] = accumulate ? out[c] + v : v;
    }
}

// ------------------------------------------------------------------ host side
bool aligned(const void* p, uintptr_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

int threads_for(int nv, int per_thread) {
    const int t = (nv + per_thread - 1) / per_thread;
    return (t + 31) / 32 * 32;
}

// Vectors of 8 a thread holds. Forward: four, which keeps the most loads in flight; fewer where a row has too few threads then.
// Rows of 2048 and shorter: two / four 80.5 / 85.5 us (32768 x 2048); up to four short rows an SM: 4.0 / 4.5 us (512 x 4096;
// 1024 x 4096: 6.9 / 5.8); a row an SM: as few as possible (one row of 4096: 512 threads). Gradient: blocks of
// 512 threads at most, which leave registers for the next row's loads: one up to 4096 elements, two up to 8192 (4096 x 8192:
// 52 us; one in blocks of 1024 threads 55), four beyond. Up to 4096 two or three smaller blocks of two vectors, with or without
// loads ahead, take the same time or longer (8192 x 4096: 49 to 71 us; as it is 49).
int fwd_vec(int rows, int H) {
    if (rows <= sm_count()) return H <= 8192 ? 1 : 2;
    return H <= 2048 || (H <= 4096 && rows <= 4 * sm_count()) ? 2 : 4;
}
constexpr int grad_vec(int H) { return H <= 4096 ? 1 : H <= 8192 ? 2 : 4; }

template <int NV, bool VEC>
int launch_forward(const NormParams& p, cudaStream_t st) {
    const int t = threads_for((p.H + 7) / 8, NV);
    // three full rounds of the resident blocks (64 registers a thread) at most: the rest of the rows is walked by the blocks.
    // Rounds of 2048 threads, 2.25 of them for 7168 elements: 81 us instead of 75 (9000 rows)
    const long long most = static_cast<long long>(sm_count()) * 3 * (1024 / t);
    const long long grid = p.rows < most ? p.rows : most;
    CF_CUDA(launch_pdl(k_add_rmsnorm<NV, VEC>, dim3(static_cast<unsigned>(grid)), dim3(t), 0, st, p));
    CF_LAUNCH_CHECK("add_rmsnorm");
    return CF_OK;
}

int grad_blocks(int rows, int H) {
    const int t = threads_for((H + 7) / 8, grad_vec(H));
    const int b = kBwdBlocks * (grad_vec(H) > 1 ? 1 : t <= 128 ? 8 : t <= 256 ? 4 : 2);
    return b < rows ? b : rows;
}

}  // namespace
}  // namespace cf

using namespace cf;

extern "C" {

int cf_add_rmsnorm_quantize_block128(const void* d_x, const void* d_residual_or_null, const void* d_scale, void* d_h_or_null,
                                     void* d_normed_or_null, float* d_rms_or_null, void* d_out8_or_null, int ld_out8, float* d_descale,
                                     long long descale_ld_row, long long descale_ld_block, int rows, int H, float eps, void* stream) {
    const char* fn = "cf_add_rmsnorm_quantize_block128";
    CF_REQUIRE(rows >= 0 && H > 0, "%s: bad shape", fn);
    if (H > kMaxH) { set_error("%s: rows of at most %d elements", fn, kMaxH); return CF_ERR_LIMIT; }
    CF_REQUIRE(eps > 0.0f, "%s: eps must be positive", fn);
    if (rows == 0) return CF_OK;
    CF_REQUIRE((d_out8_or_null != nullptr) == (d_descale != nullptr), "%s: codes and descales go together", fn);
    CF_REQUIRE(d_x && d_scale, "%s: null input", fn);
    CF_REQUIRE(d_out8_or_null || d_normed_or_null, "%s: no output", fn);
    CF_REQUIRE(d_h_or_null || !d_residual_or_null, "%s: the sum with a residual needs a buffer", fn);
    CF_REQUIRE(!d_out8_or_null || ld_out8 >= H, "%s: output pitch smaller than a row", fn);
    CF_REQUIRE(aligned(d_x, 2) && aligned(d_residual_or_null, 2) && aligned(d_scale, 2) && aligned(d_h_or_null, 2) &&
               aligned(d_normed_or_null, 2) && aligned(d_rms_or_null, 4) && aligned(d_descale, 4), "%s: misaligned pointer", fn);
    const int rc = require_sm100();
    if (rc != CF_OK) return rc;
    NormParams p = {};
    p.x = static_cast<const uint16_t*>(d_x); p.res = static_cast<const uint16_t*>(d_residual_or_null);
    p.gain = static_cast<const uint16_t*>(d_scale);
    p.h = static_cast<uint16_t*>(d_h_or_null); p.normed = static_cast<uint16_t*>(d_normed_or_null);
    p.rms = d_rms_or_null; p.out8 = static_cast<uint8_t*>(d_out8_or_null); p.ld_out8 = ld_out8;
    p.descale = d_descale; p.d_row = descale_ld_row; p.d_blk = descale_ld_block;
    p.rows = rows; p.H = H; p.eps = eps;
    p.vec8 = aligned(d_out8_or_null, 8) && ld_out8 % 8 == 0;
    const bool vec = H % 8 == 0 && aligned(d_x, 16) && aligned(d_residual_or_null, 16) && aligned(d_scale, 16) &&
                     aligned(d_h_or_null, 16) && aligned(d_normed_or_null, 16);
    cudaStream_t st = as_stream(stream);
    if (!vec) return launch_forward<4, false>(p, st);
    const int nv = fwd_vec(rows, H);
    return nv == 1 ? launch_forward<1, true>(p, st) : nv == 2 ? launch_forward<2, true>(p, st) : launch_forward<4, true>(p, st);
}

size_t cf_add_rmsnorm_backward_scratch_floats(int rows, int H) {
    if (rows <= 0 || H <= 0 || H > kMaxH) return 0;
    return static_cast<size_t>(grad_blocks(rows, H)) * H;
}

int cf_add_rmsnorm_backward(const void* d_dy, const void* d_h, const void* d_scale, const float* d_rms, const void* d_dh_or_null, void* d_dx,
                            float* d_dscale_or_null, int accumulate_dscale, float* d_scratch, size_t scratch_floats, int rows, int H,
                            void* stream) {
    const char* fn = "cf_add_rmsnorm_backward";
    CF_REQUIRE(rows >= 0 && H > 0, "%s: bad shape", fn);
    if (H > kMaxH) { set_error("%s: rows of at most %d elements", fn, kMaxH); return CF_ERR_LIMIT; }
    CF_REQUIRE(aligned(d_dscale_or_null, 4) && aligned(d_rms, 4) && aligned(d_scratch, 4), "%s: misaligned pointer", fn);
    cudaStream_t st = as_stream(stream);
    if (rows == 0) {                                    // a sum over no rows
        if (d_dscale_or_null && !accumulate_dscale) CF_CUDA(cudaMemsetAsync(d_dscale_or_null, 0, sizeof(float) * H, st));
        return CF_OK;
    }
    CF_REQUIRE(d_dy && d_h && d_scale && d_rms && d_dx, "%s: null pointer", fn);
    CF_REQUIRE(aligned(d_dy, 2) && aligned(d_h, 2) && aligned(d_scale, 2) && aligned(d_dh_or_null, 2) && aligned(d_dx, 2), "%s: misaligned pointer", fn);
    const size_t need = cf_add_rmsnorm_backward_scratch_floats(rows, H);
    if (d_dscale_or_null && (!d_scratch || scratch_floats < need)) {
        set_error("%s: %zu floats of scratch needed", fn, need);
        return CF_ERR_LIMIT;
    }
    const int rc = require_sm100();
    if (rc != CF_OK) return rc;
    NormGradParams p = {};
    p.dy = static_cast<const uint16_t*>(d_dy); p.h = static_cast<const uint16_t*>(d_h); p.gain = static_cast<const uint16_t*>(d_scale);
    p.rms = d_rms; p.dh = static_cast<const uint16_t*>(d_dh_or_null); p.dx = static_cast<uint16_t*>(d_dx);
    p.partial = d_dscale_or_null ? d_scratch : nullptr;
    p.rows = rows; p.H = H;
    const bool vec = H % 8 == 0 && aligned(d_dy, 16) && aligned(d_h, 16) && aligned(d_scale, 16) && aligned(d_dh_or_null, 16) && aligned(d_dx, 16);
    const int nv = grad_vec(H), t = threads_for((H + 7) / 8, nv), blocks = grad_blocks(rows, H);
    auto launch = [&](auto vectors) {
        constexpr int NV = decltype(vectors)::value;
        return vec ? launch_pdl(k_add_rmsnorm_grad<NV, true>, dim3(blocks), dim3(t), 0, st, p)
                   : launch_pdl(k_add_rmsnorm_grad<NV, false>, dim3(blocks), dim3(t), 0, st, p);
    };
    if (nv == 1) CF_CUDA(launch(std::integral_constant<int, 1>()));
    else if (nv == 2) CF_CUDA(launch(std::integral_constant<int, 2>()));
    else CF_CUDA(launch(std::integral_constant<int, 4>()));
    CF_LAUNCH_CHECK("add_rmsnorm_grad");
    if (d_dscale_or_null) {
        CF_CUDA(launch_pdl(k_sum_partials, dim3((H + 31) / 32), dim3(1024), 0, st, d_scratch, blocks, H, d_dscale_or_null, accumulate_dscale));
        CF_LAUNCH_CHECK("sum_partials");
    }
    return CF_OK;
}

}  // extern "C"
