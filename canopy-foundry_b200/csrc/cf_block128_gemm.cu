// Block-scaled FP8 GEMM for sm_100a.
//
//   C[m,n] = sum over blocks b of 128 along K:  da[m,b] * db[n,b] * sum_{k in b} A8[m,k] * B8[n,k]
//
// The scale changes along the contraction, so one accumulator per output cannot take the whole sum: the tensor cores
// multiply one block of 128 (four tcgen05.mma of 32) into a TMEM accumulator that starts from zero, and the epilogue
// warps fold each finished block into fp32 registers, acc += (da db) * block, while the tensor cores fill the other TMEM
// buffer with the next block. Both operands' scales are arbitrary fp32 numbers (no power-of-two restriction).
//
// Wide form (k_gemm_b128): tiles of 256 x 256 per CTA pair (cta_group::2) or 128 x 256 per CTA, persistent, 384 threads:
//   warp 0       TMA producer (one elected lane)
//   warps 1, 3   MMA issuers for even and odd blocks (one elected lane each); warp 1 owns the TMEM allocation
//   warp 2       scales: global memory -> shared-memory ring
//   warps 4..11  promotion + epilogue: each owns 32 rows x 128 columns of the CTA's 128 x 256 tile in 128 registers a thread
// Per block of 128 the MMAs of a pair take 590 clocks; the promotion's 64 packed multiply-adds a thread, from two warps on every
// scheduler, keep its fp32 pipe busy for 256 (512 where both operands' scales change inside the tile) and come with 128 KB of
// TMEM reads per CTA. The two overlap but for the hand-over: 775 clocks a block at 8192^3 (460 to 477 us at the 1.45 to 1.49 GHz
// that the power cap leaves), 1296 with a scale per column.
//
// Narrow form (k_gemm_b128_narrow): few rows of A (tokens), or too few tiles of the wide form to fill the chip. The weights take
// the MMA's 128-row side and TN tokens its column side, and the contraction is split over a cluster of CTAs whose partial sums
// meet in distributed shared memory, added in rank order: every weight byte is read once, by enough CTAs to fill the chip, and
// no atomics are involved.
//
// Every wait on an mbarrier is bounded: a wait that gives up raises an abort flag, records a code in the context's status
// word, drains the CTA's own copies and MMAs, frees TMEM and returns.
#include <atomic>

#include "cf_common.cuh"
#include "cf_internal.cuh"
#include "cf_tc.cuh"

namespace cf {

int* ctx_status(cf_ctx* c);
int ctx_device(cf_ctx* c);

namespace {

using namespace tc;

constexpr int BM = 128;                 // rows of A / C per CTA (TMEM lanes)
constexpr int BN = 256;                 // output columns per tile
constexpr int SB = 128;                 // elements of K that share a scale == BK
constexpr int NUM_THREADS = 384;        // warpgroup 0: producer, two MMA issuers, scales; warpgroups 1 and 2: promotion + epilogue
constexpr int EPI_WARPS = 8;
// Registers: the launch gives every thread kLaunchRegs; warpgroup 0 hands most of its share to the two others, which hold 128
// accumulators a thread. 40 x 128 + 232 x 256 = 168 x 384: the shares add up to what the launch has (the host checks that).
constexpr int kLaunchRegs = 168, kLeanRegs = 40, kWideRegs = 232;
static_assert(kLeanRegs * 128 + kWideRegs * 256 <= kLaunchRegs * NUM_THREADS, "register shares");
constexpr int TMEM_COLS = 512;          // two 128x256 fp32 block sums per CTA
constexpr int C_STAGING = EPI_WARPS * C_BOX_BYTES;
// Scales on their way from global memory: per stage of the operand ring the 128 row scales and the column scales (256, or one per
// 128 columns) of the block, filled by a warp of its own with 4-byte asynchronous copies as soon as the promotion has read the
// block that had the slot before. They land on the barrier that tells the block's sums are there, so the promotion waits once
// per block. A scale's first use misses L1 and often L2 (another line for every block of K): loaded by the promotion warps one
// block ahead, or copied by them several blocks ahead, the scales took more of their time than the promotion itself.
constexpr int SCALE_ENTRY = BM + BN;                       // floats

template <bool PAIR>
struct Cfg {
    static constexpr int B_ROWS = PAIR ? 128 : 256;
    static constexpr int STAGES = PAIR ? 5 : 3;
    static constexpr int A_STAGE = BM * BK;
    static constexpr int B_STAGE = B_ROWS * BK;
    static constexpr int TILE_M = PAIR ? 256 : 128;
    static constexpr int RING = STAGES * (A_STAGE + B_STAGE);
    static constexpr int SCALE_RING = STAGES * SCALE_ENTRY * 4;
    static constexpr int SMEM_BYTES = RING + C_STAGING + SCALE_RING + 1024 /*alignment slack*/ + 512 /*barriers*/;
};

enum OutKind { OUT_BF16 = 0, OUT_F32 = 1, OUT_F32_ADD = 2, OUT_BF16_ADD = 3 };

struct Params {
    int M = 0, N = 0, K = 0;                 // M: rows of C (grouped: rows of the compact buffers)
    int groups = 0;                          // 0: dense
    const int* d_counts = nullptr;
    const int* d_offsets = nullptr;
    const float* sa = nullptr;               // sa[row * sa_row + block * sa_blk]
    long long sa_row = 0, sa_blk = 0;
    const float* sb = nullptr;               // sb[(column / b_per) * sb_row + block * sb_blk + group * sb_group]
    long long sb_row = 0, sb_blk = 0, sb_group = 0;
    void* C = nullptr;
    long long ldc = 0;
    int out_kind = OUT_BF16;
    int tma_out = 0;                         // full boxes leave through TMA
    int a_mn = 0, b_mn = 0;                  // operand lies [K, rows] in memory
    int a_e5m2 = 0, b_e5m2 = 0;
    int raster_m = 8;
    int* d_status = nullptr;
};

// ---- packed fp32 pairs ----------------------------------------------------------------------------------------------
__device__ __forceinline__ uint64_t pack_f2(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpack_f2(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma_f2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul_f2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr)
        : "memory");
}
// 4 bytes from global to shared memory without a register; zero where !ok (src is then not read, but has to be an address).
__device__ __forceinline__ void cp_async4(uint32_t dst, const float* src, bool ok) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(ok ? 4 : 0) : "memory");
}
// Arrives on the barrier once this thread's earlier asynchronous copies have landed (the count includes every such thread).
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ uint16_t to_bf16_bits(float v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v)); }

__device__ __forceinline__ void store_value(const Params& p, long long row, long long col, float v) {
    const long long i = row * p.ldc + col;
    if (p.out_kind == OUT_BF16) static_cast<uint16_t*>(p.C)[i] = to_bf16_bits(v);
    else if (p.out_kind == OUT_F32) static_cast<float*>(p.C)[i] = v;
    else if (p.out_kind == OUT_F32_ADD) static_cast<float*>(p.C)[i] += v;
    else {
        uint16_t* c = static_cast<uint16_t*>(p.C) + i;
        *c = to_bf16_bits(bf16_bits_to_f32(*c) + v);
    }
}

// Frees a TMEM buffer on the leader's barrier. The default (CTA-scope) release is enough: what is handed over is TMEM, whose
// reads tcgen05.wait::ld and the tcgen05 fence have completed. A cluster-scope release costs a memory barrier that waits for
// the scale loads in flight, once per block of K.
__device__ __forceinline__ void mbar_arrive_remote(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// One lane of the (converged) warp. Inside such a branch the compiler keeps descriptors in uniform registers.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

// Ties a read's registers to this place: the read has been waited for, and what follows uses them from here on only.
__device__ __forceinline__ void pin(uint32_t (&v)[32]) {
    asm volatile("" : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]),
                 "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]),
                 "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]),
                 "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31]));
}
// ---- tiles ----------------------------------------------------------------------------------------------------------
struct Tile {
    int row0;        // first row of A / C
    int end;         // rows [row0, end) belong to the tile's group
    int n0;
    int group;
};

// Rows of a group, cut to the buffer: counts and offsets are device data, and a row outside [0, M) is never touched.
__device__ __forceinline__ void group_span(const Params& p, const int* counts, const int* offsets, int g, int& first, int& n) {
    first = offsets[g];
    n = counts[g];
    if (first < 0 || first >= p.M || n < 0) { n = 0; first = 0; }
    n = min(n, p.M - first);
}
__device__ __forceinline__ int row_blocks(const Params& p, const int* counts, const int* offsets, int TM) {
    if (p.groups == 0) return (p.M + TM - 1) / TM;
    int t = 0;
    for (int g = 0; g < p.groups; ++g) {
        int first, n;
        group_span(p, counts, offsets, g, first, n);
        t += (n + TM - 1) / TM;
    }
    return t;
}
// Bands of raster_m row blocks: consecutive tiles walk down a band, then one column block right, so the tiles in flight
// share few slabs of A and B.
__device__ __forceinline__ Tile tile_at(const Params& p, const int* counts, const int* offsets, int tile, int m_blocks, int TM) {
    Tile t;
    const int n_blocks = (p.N + BN - 1) / BN;
    const int band_tiles = p.raster_m * n_blocks;
    const int band = tile / band_tiles;
    const int first_m = band * p.raster_m;
    const int band_m = min(p.raster_m, m_blocks - first_m);
    const int r = tile - band * band_tiles;
    const int nb = r / band_m;
    int mb = first_m + (r - nb * band_m);
    t.n0 = nb * BN;
    if (p.groups == 0) {
        t.group = 0;
        t.row0 = mb * TM;
        t.end = p.M;
        return t;
    }
    int g = 0, first = 0, n = 0;
    for (; g < p.groups; ++g) {
        group_span(p, counts, offsets, g, first, n);
        const int blocks = (n + TM - 1) / TM;
        if (mb < blocks) break;
        mb -= blocks;
    }
    t.group = g;
    t.row0 = first + mb * TM;
    t.end = first + n;
    return t;
}

constexpr int kGroupsInSmem = 128;

// BVEC: db has one value per column of C and block (b_per = 1); otherwise one per 128 columns and block.
template <bool PAIR, bool BVEC>
__global__ void __launch_bounds__(NUM_THREADS, 1)
k_gemm_b128(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
            const __grid_constant__ CUtensorMap map_c, const Params p) {
    using C = Cfg<PAIR>;
    constexpr int STAGES = C::STAGES, A_STAGE = C::A_STAGE, B_STAGE = C::B_STAGE, TM = C::TILE_M;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    const uint32_t smem_a = base;
    const uint32_t smem_b = base + STAGES * A_STAGE;
    const uint32_t smem_c = smem_b + STAGES * B_STAGE;
    const uint32_t bars = smem_c + C_STAGING + C::SCALE_RING;
    // per stage: operands there; block multiplied and its scales there; scales read
    const uint32_t full_bar = bars, done_bar = bars + 8 * STAGES, sempty_bar = bars + 16 * STAGES;
    const uint32_t tempty_bar = bars + 24 * STAGES, drain_bar = tempty_bar + 16;
    uint8_t* gen = smem_raw + (base - raw);
    volatile uint32_t* s_tmem = reinterpret_cast<volatile uint32_t*>(gen + C::RING + C_STAGING + C::SCALE_RING + 24 * STAGES + 32);
    const uint32_t ring = smem_c + C_STAGING;
    const float* ring_f = reinterpret_cast<const float*>(gen + C::RING + C_STAGING);
    volatile int* s_abort = reinterpret_cast<volatile int*>(const_cast<uint32_t*>(s_tmem) + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t cta_rank = PAIR ? cluster_ctarank() : 0u;
    const bool leader = cta_rank == 0;
    const int unit = PAIR ? (blockIdx.x >> 1) : blockIdx.x;
    const int n_units = PAIR ? (gridDim.x >> 1) : gridDim.x;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full_bar + 8 * s, 1);
            mbar_init(done_bar + 8 * s, 1 + 32);             // the commit, and the lanes of the scale warp as their copies land
            mbar_init(sempty_bar + 8 * s, EPI_WARPS);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(tempty_bar + 8 * a, PAIR ? 2 * EPI_WARPS : EPI_WARPS);
            mbar_init(drain_bar + 8 * a, 1);
        }
        s_abort[0] = 0;
        s_abort[1] = 0;                                      // stays 0: abort source for the drain waits
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_b) : "memory");
        if (p.tma_out) asm volatile("prefetch.tensormap [%0];" ::"l"(&map_c) : "memory");
    }
    if (warp == 1) {
        if (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(const_cast<uint32_t*>(s_tmem))), "r"(TMEM_COLS) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(const_cast<uint32_t*>(s_tmem))), "r"(TMEM_COLS) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    tcgen05_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync_all();
    tcgen05_fence_after();
    const uint32_t tmem_base = *s_tmem;
    pdl_wait();                                              // everything above touched only this CTA's own memory

    __shared__ int s_groups[2 * kGroupsInSmem];
    const int* counts = p.d_counts;
    const int* offsets = p.d_offsets;
    if (p.groups > 0 && p.groups <= kGroupsInSmem) {         // the tile mapping walks them for every tile
        for (int e = threadIdx.x; e < p.groups; e += NUM_THREADS) {
            s_groups[e] = p.d_counts[e];
            s_groups[kGroupsInSmem + e] = p.d_offsets[e];
        }
        __syncthreads();
        counts = s_groups;
        offsets = s_groups + kGroupsInSmem;
    }
    const int m_blocks = row_blocks(p, counts, offsets, TM);
    const int total_tiles = m_blocks * ((p.N + BN - 1) / BN);
    const int k_iters = (p.K + BK - 1) / BK;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLeanRegs));
    if (warp == 0) {
        // ------------------------------------------------------------ TMA producer (both CTAs of a pair)
        if (lane == 0) {
            int it = 0, s = 0;
            uint32_t phase = 1;                              // the ring starts out empty
            bool ok = true;
            const uint32_t full_dst = PAIR ? mapa(full_bar, 0) : full_bar;
            for (int tile = unit; ok && tile < total_tiles; tile += n_units) {
                const Tile tc_ = tile_at(p, counts, offsets, tile, m_blocks, TM);
                const int a_row = tc_.row0 + static_cast<int>(cta_rank) * BM;
                const int b_col = tc_.n0 + static_cast<int>(cta_rank) * C::B_ROWS;       // rank is 0 in the single form
                for (int kb = 0; kb < k_iters; ++kb, ++it) {
                    if (!mbar_wait(done_bar + 8 * s, phase, s_abort)) { ok = false; break; }
                    // K-major operand: x runs along K. MN-major operand ([K, rows] in memory): x runs along the rows, the
                    // box rows are K (pair form only: a CTA's share is one box of 128 bytes)
                    const int ax = p.a_mn ? a_row : kb * BK, ay = p.a_mn ? kb * BK : a_row;
                    const int bx = p.b_mn ? b_col : kb * BK, by = p.b_mn ? kb * BK : tc_.group * p.N + b_col;
                    if (PAIR) {
                        if (leader) mbar_expect_tx(full_bar + 8 * s, 2 * (A_STAGE + B_STAGE));
                        tma_load_2d_pair(smem_a + s * A_STAGE, &map_a, full_dst + 8 * s, ax, ay);
                        tma_load_2d_pair(smem_b + s * B_STAGE, &map_b, full_dst + 8 * s, bx, by);
                    } else {
                        mbar_expect_tx(full_bar + 8 * s, A_STAGE + B_STAGE);
                        tma_load_2d(smem_a + s * A_STAGE, &map_a, full_bar + 8 * s, ax, ay);
                        tma_load_2d(smem_b + s * B_STAGE, &map_b, full_bar + 8 * s, bx, by);
                    }
                    if (++s == STAGES) { s = 0; phase ^= 1u; }
                }
            }
            if (!ok && !*s_abort) { *s_abort = 1; atomicExch(p.d_status, 0x500 | 1); }
            if ((*s_abort || !ok) && leader) {
                for (int j = max(0, it - STAGES); j < it; ++j)
                    mbar_wait(full_bar + 8 * (j % STAGES), (j / STAGES) & 1, s_abort + 1 /*never set*/, DRAIN_NS);
            }
        }
    } else if (warp == 1 || warp == 3) {
        // ------------------------------------------------------------ MMA issuers (leader CTA only)
        // Warp 1 issues the even blocks, warp 3 the odd ones, each into its own TMEM buffer: the two sequences do not depend on
        // each other, and while one warp waits for barriers and commits, the other one's MMAs keep the tensor cores fed. One
        // issuer for both left them idle for half of the time (1030 clocks a block where its MMAs take 590). The warps stay
        // converged and one elected lane issues: descriptors then live in uniform registers, and a block's four MMAs and the
        // commit take 160 clocks to issue instead of 520 from a lane of its own.
        if (leader) {
            const bool elected = elect_one();
            const int mine = warp >> 1;                      // 0: even, 1: odd
            const int blocks = unit < total_tiles ? ((total_tiles - unit - 1) / n_units + 1) * k_iters : 0;
            const uint32_t idesc = make_idesc(p.a_e5m2, p.b_e5m2, TM, BN, p.a_mn, p.b_mn);
            // one MMA covers 32 of K: 32 bytes further inside the swizzle atom of a K-major operand, 32 rows of 128 bytes
            // further in an MN-major one
            const uint32_t a_step = p.a_mn ? 256u : 2u, b_step = p.b_mn ? 256u : 2u;
            const uint32_t tmem_d = tmem_base + mine * BN, tempty = tempty_bar + 8 * mine;
            const uint64_t desc_a0 = make_smem_desc(smem_a), desc_b0 = make_smem_desc(smem_b);
            int s = mine;
            uint32_t phase = 0, t_phase = 1;
            bool ok = true;
            for (int it = mine; it < blocks; it += 2) {
                const uint64_t adesc = desc_a0 + static_cast<uint32_t>(s * (A_STAGE >> 4));
                const uint64_t bdesc = desc_b0 + static_cast<uint32_t>(s * (B_STAGE >> 4));
                if (elected && ok) {                         // a wait that gave up: the loop runs out without doing anything
                    ok = mbar_wait(tempty, t_phase, s_abort) && mbar_wait(full_bar + 8 * s, phase, s_abort);
                    if (ok) {
                        tcgen05_fence_after();
#pragma unroll
                        for (int kk = 0; kk < BK / UMMA_K; ++kk) {
                            if (PAIR) umma_f8_pair(tmem_d, adesc + a_step * kk, bdesc + b_step * kk, idesc, kk != 0 ? 1u : 0u);
                            else umma_f8(tmem_d, adesc + a_step * kk, bdesc + b_step * kk, idesc, kk != 0 ? 1u : 0u);
                        }
                        // the stage may be filled again, and the block's sums may be read (in both CTAs of a pair)
                        if (PAIR) tcgen05_commit_pair(done_bar + 8 * s); else tcgen05_commit(done_bar + 8 * s);
                    }
                }
                __syncwarp();
                t_phase ^= 1u;
                s += 2;
                if (s >= STAGES) { s -= STAGES; phase ^= 1u; }
            }
            if (!ok && elected && !*s_abort) { *s_abort = 1; atomicExch(p.d_status, 0x600 | 1); }
            __syncwarp();
            if ((*s_abort || !ok) && elected) {
                if (PAIR) asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(drain_bar + 8 * mine) : "memory");
                else tcgen05_commit(drain_bar + 8 * mine);
                mbar_wait(drain_bar + 8 * mine, 0, s_abort + 1, DRAIN_NS);
            }
        }
    } else if (warp == 2) {
        // ------------------------------------------------------------ scales (both CTAs of a pair, their own rows)
        int e = 0;
        uint32_t phase = 1;                                  // the ring starts out empty
        bool ok = true;
        for (int tile = unit; ok && tile < total_tiles; tile += n_units) {
            const Tile tc_ = tile_at(p, counts, offsets, tile, m_blocks, TM);
            const int row = tc_.row0 + static_cast<int>(cta_rank) * BM + lane;
            const float* sa = p.sa + row * p.sa_row;
            const float* sb = p.sb + tc_.group * p.sb_group + (BVEC ? (tc_.n0 + lane) * p.sb_row : (tc_.n0 / SB + lane) * p.sb_row);
            for (int kb = 0; kb < k_iters; ++kb) {
                if (!mbar_wait(sempty_bar + 8 * e, phase, s_abort)) { ok = false; break; }
                const uint32_t dst = ring + e * (SCALE_ENTRY * 4) + lane * 4;
                // rows and columns outside of the product get scale 0 (their results are not stored)
#pragma unroll
                for (int q = 0; q < BM / 32; ++q) {
                    const bool in = row + 32 * q < tc_.end;
                    cp_async4(dst + 128 * q, in ? sa + 32 * q * p.sa_row : p.sa, in);
                }
                if (BVEC) {
#pragma unroll
                    for (int q = 0; q < BN / 32; ++q) {
                        const bool in = tc_.n0 + lane + 32 * q < p.N;
                        cp_async4(dst + 4 * BM + 128 * q, in ? sb + 32 * q * p.sb_row : p.sb, in);
                    }
                } else if (lane < BN / SB) {
                    const bool in = tc_.n0 + lane * SB < p.N;
                    cp_async4(dst + 4 * BM, in ? sb : p.sb, in);
                }
                cp_async_arrive(done_bar + 8 * e);
                sa += p.sa_blk;
                sb += p.sb_blk;
                if (++e == STAGES) { e = 0; phase ^= 1u; }
            }
        }
        if (!ok && lane == 0 && !*s_abort) { *s_abort = 1; atomicExch(p.d_status, 0xb00 | 1); }
        cp_async_wait_all();
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kWideRegs));
        // ------------------------------------------------------------ promotion + epilogue (both CTAs of a pair)
        const int quarter = warp & 3;                      // TMEM lanes this warp may read
        const int half = (warp - 4) >> 2;                  // which 128 columns of the tile
        const uint32_t tempty_dst = PAIR ? mapa(tempty_bar, 0) : tempty_bar;
        const uint32_t box = smem_c + static_cast<uint32_t>(warp - 4) * C_BOX_BYTES;
        float* box_f = reinterpret_cast<float*>(gen + C::RING + (warp - 4) * C_BOX_BYTES);
        const uint64_t store_policy = l2_policy_evict_first();
        int it = 0, st = 0;                                // block, its stage
        uint32_t d_phase = 0;
        bool ok = true;                                    // per lane: one whose wait gave up goes on without waiting, so that the
                                                           // warp stays together (the results are reported as invalid)
        for (int tile = unit; tile < total_tiles; tile += n_units) {
            const Tile tc_ = tile_at(p, counts, offsets, tile, m_blocks, TM);
            const int warp_row = tc_.row0 + static_cast<int>(cta_rank) * BM + quarter * 32;
            const int wcol = tc_.n0 + half * 128;          // first column of this warp
            uint64_t acc[64];
#pragma unroll
            for (int j = 0; j < 64; ++j) acc[j] = 0ull;
            // The reads of TMEM run one chunk of 32 columns ahead of the arithmetic, over block boundaries too: while a chunk
            // is folded in, the next one is on its way. A buffer goes back as soon as its last chunk is in registers.
            const uint32_t tcol = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + half * 128;
            uint32_t v[2][32];
            ok = ok && mbar_wait(done_bar + 8 * st, d_phase, s_abort);
            tcgen05_fence_after();
            tmem_ld32(tcol + (it & 1) * BN, v[0]);
            for (int kb = 0; kb < k_iters; ++kb) {
                const int buf = it & 1;
                const float* entry = ring_f + st * SCALE_ENTRY;
                const float* cs = entry + BM + half * 128;
                const float s_row = BVEC ? entry[quarter * 32 + lane] : entry[quarter * 32 + lane] * entry[BM + half];
                const uint64_t s2 = pack_f2(s_row, s_row);
                const uint32_t done = sempty_bar + 8 * st;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    tmem_ld_wait();
                    if (c < 3) {
                        tmem_ld32(tcol + buf * BN + (c + 1) * 32, v[(c + 1) & 1]);
                    } else {
                        tcgen05_fence_before();
                        __syncwarp();
                        if (lane == 0) {
                            if (PAIR) mbar_arrive_remote(tempty_dst + 8 * buf); else mbar_arrive(tempty_bar + 8 * buf);
                            if (!BVEC) mbar_arrive(done);
                        }
                        ++it;
                        if (++st == STAGES) { st = 0; d_phase ^= 1u; }
                        if (kb + 1 < k_iters) {
                            ok = ok && mbar_wait(done_bar + 8 * st, d_phase, s_abort);
                            tcgen05_fence_after();
                            tmem_ld32(tcol + (it & 1) * BN, v[0]);
                        }
                    }
                    pin(v[c & 1]);
#pragma unroll
                    for (int j = 0; j < 16; j += 2) {
                        uint64_t x0 = pack_f2(__uint_as_float(v[c & 1][2 * j]), __uint_as_float(v[c & 1][2 * j + 1]));
                        uint64_t x1 = pack_f2(__uint_as_float(v[c & 1][2 * j + 2]), __uint_as_float(v[c & 1][2 * j + 3]));
                        if (BVEC) {
                            const ulonglong2 b4 = *reinterpret_cast<const ulonglong2*>(cs + c * 32 + 2 * j);
                            x0 = mul_f2(x0, b4.x);
                            x1 = mul_f2(x1, b4.y);
                        }
                        acc[c * 16 + j] = fma_f2(x0, s2, acc[c * 16 + j]);
                        acc[c * 16 + j + 1] = fma_f2(x1, s2, acc[c * 16 + j + 1]);
                    }
                }
                if (BVEC) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(done);
                }
            }
            // ---- the tile's 32 rows x 128 columns of this warp leave
            const bool f32 = p.out_kind == OUT_F32 || p.out_kind == OUT_F32_ADD;
            // a box may only leave whole: in the ragged form its rows must all belong to the group
            const bool boxes = p.tma_out && warp_row < tc_.end && (p.groups == 0 || warp_row + 32 <= tc_.end);
            const uint32_t row_off = static_cast<uint32_t>(lane) * 128u;
            const uint32_t sw = static_cast<uint32_t>(lane & 7);
            if (lane == 0) bulk_wait_read_0();
            __syncwarp();
#pragma unroll
            for (int c = 0; c < 4; ++c) {                  // 32 columns at a time
                const int col0 = wcol + c * 32;
                const int width = f32 ? 32 : 64;
                const int box_col = f32 ? col0 : wcol + (c >> 1) * 64;
                if (col0 < p.N) {                          // warp-uniform
                    if (boxes && box_col + width <= p.N) {
                        if (f32 ? c > 0 : c == 2) {        // the previous box has left this buffer
                            if (lane == 0) bulk_wait_read_0();
                            __syncwarp();
                        }
                        if (f32) {
#pragma unroll
                            for (int q = 0; q < 8; ++q) {  // 16-byte chunk q of a row sits at q ^ (row % 8): 128B swizzle
                                float f[4];
                                unpack_f2(acc[c * 16 + 2 * q], f[0], f[1]);
                                unpack_f2(acc[c * 16 + 2 * q + 1], f[2], f[3]);
                                st_shared_v4(box + row_off + ((static_cast<uint32_t>(q) ^ sw) << 4), __float_as_uint(f[0]),
                                             __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
                            }
                        } else {
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                uint32_t w[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    float lo, hi;
                                    unpack_f2(acc[c * 16 + 4 * q + e], lo, hi);
                                    w[e] = pack_bf16x2(lo, hi);
                                }
                                st_shared_v4(box + row_off + ((static_cast<uint32_t>((c & 1) * 4 + q) ^ sw) << 4), w[0], w[1], w[2], w[3]);
                            }
                        }
                        if (f32 || (c & 1)) {
                            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                            __syncwarp();
                            if (lane == 0) {
                                if (p.out_kind == OUT_F32_ADD) tma_reduce_add_2d(&map_c, box, box_col, warp_row);
                                else tma_store_2d(&map_c, box, box_col, warp_row, store_policy);
                                bulk_commit();
                            }
                        }
                    } else {
                        // edges, ragged rows, unaligned or accumulated bf16 outputs: the 32 x 32 values turn around in the
                        // box, so that a warp writes 32 neighbouring columns of one row at a time
                        if (lane == 0) bulk_wait_read_0();
                        __syncwarp();
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            float lo, hi;
                            unpack_f2(acc[c * 16 + j], lo, hi);
                            box_f[lane * 32 + ((2 * j) ^ lane)] = lo;
                            box_f[lane * 32 + ((2 * j + 1) ^ lane)] = hi;
                        }
                        __syncwarp();
                        const int rows = min(32, tc_.end - warp_row);
                        for (int r = 0; r < rows; ++r)
                            if (col0 + lane < p.N) store_value(p, warp_row + r, col0 + lane, box_f[r * 32 + (lane ^ r)]);
                        __syncwarp();
                    }
                }
            }
        }
        if (lane == 0) bulk_wait_all();
        if (!ok && !*s_abort) { *s_abort = 1; atomicExch(p.d_status, 0x700 | 1); }
    }

    tcgen05_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync_all();          // the peer may still read this CTA's operands / signal its barriers
    if (warp == 1) {
        __syncwarp();
        tcgen05_fence_after();
        if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
    }
}

// ------------------------------------------------------------------ narrow form
constexpr int NARROW_THREADS = 192;        // warp 0 producer, warp 1 MMA issuer, warps 2..5 promotion
template <int TN>
struct Narrow {
    static constexpr int W_STAGE = 128 * BK;
    static constexpr int X_STAGE = TN * BK;
    static constexpr int STAGES = TN <= 32 ? 5 : 4;
    static constexpr int RING = STAGES * (W_STAGE + X_STAGE);
    static constexpr int AHEAD = 4;                        // blocks whose scales are on their way
    // per promotion warp: AHEAD entries of TN token scales and a weight scale per lane, two copies of the products in use
    static constexpr int WARP_SCALES = AHEAD * (TN + 32) + 2 * TN;
    static constexpr int SCALES = 4 * WARP_SCALES * 4;
    static constexpr int TMEM = 2 * TN < 32 ? 32 : 2 * TN;
    static constexpr int PARTIAL = TN * 128 * 4;           // overlays the ring after the last block
    static constexpr int SMEM_BYTES = RING + SCALES + 1024 + 256;
    static_assert(PARTIAL <= RING, "partial sums overlay the ring");
};

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

// The partial sums part[token][128 features] of the SPLITS CTAs of a cluster, added in rank order and stored. Four features a
// thread, all ranks' loads of an item in flight at once: one load after the other (250 clocks each out of another SM) took
// longer than the product itself, 10.4 us instead of 9.5 for 64 x 4096 x 4096 split eight ways.
template <int SPLITS>
__device__ __forceinline__ void join_partials(const Params& p, uint32_t part, int tokens, int rank, int m0, int n0, int vec) {
    uint32_t base[SPLITS];
#pragma unroll
    for (int r = 0; r < SPLITS; ++r) base[r] = SPLITS == 1 ? part : mapa(part, r);
#pragma unroll 4
    for (int i = rank * NARROW_THREADS + threadIdx.x; i < tokens * 32; i += SPLITS * NARROW_THREADS) {
        float4 v[SPLITS];
#pragma unroll
        for (int r = 0; r < SPLITS; ++r) v[r] = ld_cluster_f4(base[r] + i * 16);
#pragma unroll
        for (int r = 1; r < SPLITS; ++r) {
            v[0].x += v[r].x; v[0].y += v[r].y; v[0].z += v[r].z; v[0].w += v[r].w;
        }
        const int m = m0 + i / 32, n = n0 + (i % 32) * 4;
        if (vec && n + 4 <= p.N) {                           // bf16, stored, 8-byte aligned
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.C) + m * p.ldc + n) =
                make_uint2(pack_bf16x2(v[0].x, v[0].y), pack_bf16x2(v[0].z, v[0].w));
        } else {
            const float f[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (n + e < p.N) store_value(p, m, n + e, f[e]);
        }
    }
}

// map_w: weights [N, K]; map_x: tokens [M, K]. Grid: x = n tile * splits + rank in the cluster, y = token tile.
// BVEC: every weight row has its own scale (folded in per lane); otherwise the tile's 128 rows share one, which is multiplied
// into the token scales before they are spread.
template <int TN, bool BVEC>
__global__ void __launch_bounds__(NARROW_THREADS)
k_gemm_b128_narrow(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Params p, int splits) {
    using C = Narrow<TN>;
    constexpr int STAGES = C::STAGES;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (base - raw);
    const uint32_t smem_w = base, smem_x = base + STAGES * C::W_STAGE;
    float* s_scales = reinterpret_cast<float*>(gen + C::RING);
    const uint32_t bars = base + C::RING + C::SCALES;
    const uint32_t full_bar = bars, empty_bar = bars + 8 * STAGES, tfull_bar = bars + 16 * STAGES, tempty_bar = tfull_bar + 16,
                   drain_bar = tempty_bar + 16;
    volatile uint32_t* s_tmem = reinterpret_cast<volatile uint32_t*>(gen + C::RING + C::SCALES + 16 * STAGES + 48);
    volatile int* s_abort = reinterpret_cast<volatile int*>(const_cast<uint32_t*>(s_tmem) + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x % splits;
    const int n0 = (blockIdx.x / splits) * 128;
    const int m0 = blockIdx.y * TN;
    const int k_iters = (p.K + BK - 1) / BK;
    const int kb0 = static_cast<int>(static_cast<long long>(k_iters) * rank / splits);
    const int kb1 = static_cast<int>(static_cast<long long>(k_iters) * (rank + 1) / splits);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full_bar + 8 * s, 1);
            mbar_init(empty_bar + 8 * s, 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(tfull_bar + 8 * a, 1);
            mbar_init(tempty_bar + 8 * a, 4);
        }
        mbar_init(drain_bar, 1);
        s_abort[0] = 0;
        s_abort[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(const_cast<uint32_t*>(s_tmem))), "r"(C::TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem_base = *s_tmem;
    pdl_wait();

    uint64_t acc[TN / 2];                  // lane = output feature, pairs of tokens
#pragma unroll
    for (int j = 0; j < TN / 2; ++j) acc[j] = 0ull;

    if (warp == 0) {
        if (lane == 0) {
            bool ok = true;
            int it = 0;
            for (int kb = kb0; kb < kb1; ++kb, ++it) {
                const int s = it % STAGES;
                if (!mbar_wait(empty_bar + 8 * s, ((it / STAGES) & 1) ^ 1, s_abort)) { ok = false; break; }
                mbar_expect_tx(full_bar + 8 * s, C::W_STAGE + C::X_STAGE);
                tma_load_2d(smem_w + s * C::W_STAGE, &map_w, full_bar + 8 * s, kb * BK, n0);
                tma_load_2d(smem_x + s * C::X_STAGE, &map_x, full_bar + 8 * s, kb * BK, m0);
            }
            if (!ok && !*s_abort) { *s_abort = 1; atomicExch(p.d_status, 0x800 | 1); }
            if (*s_abort || !ok)
                for (int j = max(0, it - STAGES); j < it; ++j)
                    mbar_wait(full_bar + 8 * (j % STAGES), (j / STAGES) & 1, s_abort + 1, DRAIN_NS);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint32_t idesc = make_idesc(p.b_e5m2, p.a_e5m2, 128, TN, 0, 0);
            bool ok = true;
            int it = 0;
            for (int kb = kb0; kb < kb1; ++kb, ++it) {
                const int s = it % STAGES, buf = it & 1;
                if (!mbar_wait(tempty_bar + 8 * buf, ((it >> 1) & 1) ^ 1, s_abort)) { ok = false; break; }
                if (!mbar_wait(full_bar + 8 * s, (it / STAGES) & 1, s_abort)) { ok = false; break; }
                tcgen05_fence_after();
                const uint64_t wdesc = make_smem_desc(smem_w + s * C::W_STAGE);
                const uint64_t xdesc = make_smem_desc(smem_x + s * C::X_STAGE);
#pragma unroll
                for (int kk = 0; kk < BK / UMMA_K; ++kk)
                    umma_f8(tmem_base + buf * TN, wdesc + 2 * kk, xdesc + 2 * kk, idesc, kk != 0 ? 1u : 0u);
                tcgen05_commit(empty_bar + 8 * s);
                tcgen05_commit(tfull_bar + 8 * buf);
            }
            if (!ok && !*s_abort) { *s_abort = 1; atomicExch(p.d_status, 0x900 | 1); }
            if (*s_abort || !ok) {
                tcgen05_commit(drain_bar);
                mbar_wait(drain_bar, 0, s_abort + 1, DRAIN_NS);
            }
        }
    } else {
        // lane = output feature n, TMEM column = token
        const int quarter = warp & 3;
        const int n = n0 + quarter * 32 + lane;
        // the tile's one scale, for every lane (each multiplies it into some of the tokens' scales), or the lane's own row's
        const bool w_ok = !BVEC || n < p.N;
        const float* sw = p.sb + (w_ok ? (BVEC ? n : n0 / SB) * p.sb_row : 0) + kb0 * p.sb_blk;
        constexpr int PER = (TN + 31) / 32, ENTRY = TN + 32;
        float* ring_f = s_scales + (warp - 2) * C::WARP_SCALES;
        float* sc = ring_f + C::AHEAD * ENTRY;
        const uint32_t ring = smem_u32(ring_f) + lane * 4;
        int f_kb = kb0, f_slot = 0;
        // every lane copies what it will read itself: no barrier between the copy and its use
        auto fetch = [&]() {
            if (f_kb < kb1) {
                const uint32_t dst = ring + f_slot * (ENTRY * 4);
#pragma unroll
                for (int q = 0; q < PER; ++q) {
                    const int m = lane + 32 * q;
                    const bool in = m < TN && m0 + m < p.M;
                    if (m < TN) cp_async4(dst + 128 * q, in ? p.sa + (m0 + m) * p.sa_row + f_kb * p.sa_blk : p.sa, in);
                }
                cp_async4(dst + 4 * TN, sw, w_ok);
                if (w_ok) sw += p.sb_blk;
                ++f_kb;
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            if (++f_slot == C::AHEAD) f_slot = 0;
        };
        for (int i = 0; i < C::AHEAD; ++i) fetch();
        bool ok = true;
        int it = 0, slot = 0;
        for (int kb = kb0; kb < kb1; ++kb, ++it) {
            const int buf = it & 1;
            asm volatile("cp.async.wait_group %0;" ::"n"(C::AHEAD - 1) : "memory");
            const float w = ring_f[slot * ENTRY + TN + lane];
#pragma unroll
            for (int q = 0; q < PER; ++q)
                if (lane + 32 * q < TN) sc[buf * TN + lane + 32 * q] = ring_f[slot * ENTRY + lane + 32 * q] * (BVEC ? 1.0f : w);
            __syncwarp();
            if (++slot == C::AHEAD) slot = 0;
            fetch();
            ok = ok && mbar_wait(tfull_bar + 8 * buf, (it >> 1) & 1, s_abort);     // see the wide form
            tcgen05_fence_after();
            const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + buf * TN;
            const uint64_t w2 = pack_f2(w, w);
            constexpr int CH = TN < 32 ? 16 : 32;          // columns per read, the next one on its way while one is folded in
            uint32_t v[2][32];
            if (CH == 32) tmem_ld32(taddr, v[0]); else tmem_ld16(taddr, reinterpret_cast<uint32_t(&)[16]>(v[0]));
#pragma unroll
            for (int c = 0; c < TN / CH; ++c) {
                tmem_ld_wait();
                if (c + 1 < TN / CH) {
                    tmem_ld32(taddr + (c + 1) * 32, v[(c + 1) & 1]);
                } else {                                   // the block is in registers: its buffer goes back
                    tcgen05_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(tempty_bar + 8 * buf);
                }
#pragma unroll
                for (int j = 0; j < CH / 4; ++j) {
                    const ulonglong2 s4 = *reinterpret_cast<const ulonglong2*>(sc + buf * TN + c * CH + 4 * j);
                    uint64_t x0 = pack_f2(__uint_as_float(v[c & 1][4 * j]), __uint_as_float(v[c & 1][4 * j + 1]));
                    uint64_t x1 = pack_f2(__uint_as_float(v[c & 1][4 * j + 2]), __uint_as_float(v[c & 1][4 * j + 3]));
                    if (BVEC) { x0 = mul_f2(x0, w2); x1 = mul_f2(x1, w2); }
                    acc[(c * CH) / 2 + 2 * j] = fma_f2(x0, s4.x, acc[(c * CH) / 2 + 2 * j]);
                    acc[(c * CH) / 2 + 2 * j + 1] = fma_f2(x1, s4.y, acc[(c * CH) / 2 + 2 * j + 1]);
                }
            }
        }
        cp_async_wait_all();
        if (!ok && !*s_abort) { *s_abort = 1; atomicExch(p.d_status, 0xa00 | 1); }
    }

    tcgen05_fence_before();
    __syncthreads();                       // every block of this CTA has been consumed: the ring is free
    if (warp == 1) {
        __syncwarp();
        tcgen05_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(C::TMEM) : "memory");
    }
    float* part = reinterpret_cast<float*>(gen);                 // [TN][128]
    if (warp >= 2) {
        const int f = (warp & 3) * 32 + lane;
#pragma unroll
        for (int t = 0; t < TN; t += 2) unpack_f2(acc[t / 2], part[t * 128 + f], part[(t + 1) * 128 + f]);
    }
    const int tokens = min(TN, p.M - m0);
    const int vec = p.out_kind == OUT_BF16 && p.ldc % 4 == 0 && reinterpret_cast<uintptr_t>(p.C) % 8 == 0;
    if (splits == 1) {
        __syncthreads();
        join_partials<1>(p, base, tokens, 0, m0, n0, vec);
        return;
    }
    cluster_sync_all();
    if (splits == 2) join_partials<2>(p, base, tokens, rank, m0, n0, vec);
    else if (splits == 4) join_partials<4>(p, base, tokens, rank, m0, n0, vec);
    else join_partials<8>(p, base, tokens, rank, m0, n0, vec);
    cluster_sync_all();                                          // the others have read this CTA's sums
}

// ------------------------------------------------------------------ host side
bool aligned(const void* p, uintptr_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }
long long cdiv(long long a, long long b) { return (a + b - 1) / b; }

template <class K>
int check_regs(K* kernel) {
    cudaFuncAttributes a;
    CF_CUDA(cudaFuncGetAttributes(&a, kernel));
    if (a.numRegs < kLaunchRegs) {          // the warpgroups' shares would not add up: setmaxnreg.inc would wait for ever
        set_error("k_gemm_b128 was built with %d registers a thread, its register split needs %d", a.numRegs, kLaunchRegs);
        return CF_ERR_UNSUPPORTED;
    }
    return CF_OK;
}
template <bool PAIR>
int set_smem() {
    int rc = check_regs(k_gemm_b128<PAIR, false>);
    if (rc == CF_OK) rc = check_regs(k_gemm_b128<PAIR, true>);
    if (rc != CF_OK) return rc;

    cudaError_t e = cudaFuncSetAttribute(k_gemm_b128<PAIR, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<PAIR>::SMEM_BYTES);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k_gemm_b128<PAIR, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<PAIR>::SMEM_BYTES);
    return e == cudaSuccess ? CF_OK : cuda_fail(e, "cudaFuncSetAttribute(k_gemm_b128)");
}

// CTA pairs the current device keeps resident at once, asked once per device.
int resident_pairs(int* pairs) {
    static std::mutex mu;
    static int cached[64];                  // 0 unknown, else pairs + 1
    int dev = 0;
    CF_CUDA(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lk(mu);
    int& c = cached[dev & 63];
    if (c == 0) {
        int rc = set_smem<true>();
        if (rc == CF_OK) rc = set_smem<false>();
        if (rc != CF_OK) return rc;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(2 * sm_count());
        cfg.blockDim = dim3(NUM_THREADS);
        cfg.dynamicSmemBytes = Cfg<true>::SMEM_BYTES;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = 2; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        int n = 0;
        CF_CUDA(cudaOccupancyMaxActiveClusters(&n, k_gemm_b128<true, true>, &cfg));
        if (n < 1) { set_error("no CTA pair fits this device"); return CF_ERR_UNSUPPORTED; }
        c = n + 1;
    }
    *pairs = c - 1;
    return CF_OK;
}

template <int TN, bool BVEC>
int launch_narrow(const CUtensorMap& map_w, const CUtensorMap& map_x, const Params& p, int splits, cudaStream_t st) {
    using C = Narrow<TN>;
    static std::atomic<int> ready[64];      // the attribute is set once per device (any thread may do it)
    int dev = 0;
    CF_CUDA(cudaGetDevice(&dev));
    if (!ready[dev & 63].load(std::memory_order_acquire)) {
        CF_CUDA(cudaFuncSetAttribute(k_gemm_b128_narrow<TN, BVEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES));
        ready[dev & 63].store(1, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(cdiv(p.N, 128) * splits), static_cast<unsigned>(cdiv(p.M, TN)));
    cfg.blockDim = dim3(NARROW_THREADS);
    cfg.dynamicSmemBytes = C::SMEM_BYTES;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = splits; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    CF_CUDA(cudaLaunchKernelEx(&cfg, k_gemm_b128_narrow<TN, BVEC>, map_w, map_x, p, splits));
    CF_LAUNCH_CHECK("gemm_b128_narrow");
    return CF_OK;
}
template <int TN>
int launch_narrow_any(const CUtensorMap& map_w, const CUtensorMap& map_x, const Params& p, int splits, int b_per, cudaStream_t st) {
    return b_per == 1 ? launch_narrow<TN, true>(map_w, map_x, p, splits, st) : launch_narrow<TN, false>(map_w, map_x, p, splits, st);
}

// a_rows_mem / b_rows_mem: row extents of the two byte matrices in memory. b_per: columns of C per B scale (128 or 1).
int launch_b128(const char* fn, cf_ctx* ctx, const void* A, long long lda, const void* B, long long ldb, long long b_rows_mem, Params p, int b_per,
                cudaStream_t st) {
    if (!aligned(A, 16) || !aligned(B, 16) || lda % 16 != 0 || ldb % 16 != 0) {
        set_error("%s: the FP8 operands need 16-byte aligned bases and row pitches", fn);
        return CF_ERR_UNSUPPORTED;
    }
    int rc = require_sm100();
    if (rc != CF_OK) return rc;
    int dev = 0;
    CF_CUDA(cudaGetDevice(&dev));
    CF_REQUIRE(dev == ctx_device(ctx), "%s: the context belongs to device %d, the current device is %d", fn, ctx_device(ctx), dev);
    p.d_status = ctx_status(ctx);
    CUtensorMap map_a, map_b, map_c;
    int pairs = 0;
    rc = resident_pairs(&pairs);
    if (rc != CF_OK) return rc;
    const int k_iters = static_cast<int>(cdiv(p.K, BK));
    // CTA pairs or single CTAs: whichever is expected to end first. A block of K takes a pair's tile about 0.55 us, a single CTA's
    // (half of it) 0.58 with the chip full and 0.47 with less: the promotion sets the pace of both, so what decides is how the
    // tiles fill the last round. Ragged groups end in half a row block each on average. Measured pair / single: eight ragged
    // experts, 4096 rows x 4096 x 14336: 331 / 272 us; 1531 x 4104 x 5416: 48 / 60; 8192^3: 522 / 560.
    const int sms = sm_count();
    auto tile_count = [&](int tm) { return (p.groups > 0 ? p.M / tm + (p.groups + 1) / 2 : cdiv(p.M, tm)) * cdiv(p.N, BN); };
    const long long singles = tile_count(128);
    const long long pair_cost = cdiv(tile_count(256), pairs) * 55, single_cost = cdiv(singles, sms) * (singles <= sms ? 47 : 58);
    const bool pair = p.a_mn || p.b_mn || pair_cost <= single_cost;
    if (p.groups == 0 && !p.a_mn && !p.b_mn) {
        // The narrow form where it is expected to end before either. Its CTAs (two on an SM) take about 0.70 us per block of K; up
        // to 64 rows it reads every weight once and runs at the memory's rate.
        // Narrow / wide us, N x K: 28672 x 4096: M = 32 21.7 / 25.4, 64 24.3 / 25.6, 96 45 / 26; 4096 x 14336: 64 16.7 / 56,
        // 256 42 / 56, 384 77 / 56; 4096 x 4096: 128 10.9 / 19.6, 256 15.5 / 19.8, 384 24 / 20; 1024 x 4096: 512 10.9 / 21.
        const int tn = p.M <= 16 ? 16 : p.M <= 32 ? 32 : 64;
        const long long ctas = cdiv(p.N, 128) * cdiv(p.M, tn), room = 2ll * sms;
        int splits = 1;
        while (splits < 8 && ctas * splits * 2 <= room && k_iters >= 4 * splits) splits *= 2;
        const long long narrow_cost = cdiv(ctas * splits, room) * cdiv(k_iters, splits) * 70;
        if (p.M <= 64 || narrow_cost < (pair ? pair_cost : single_cost) * k_iters) {
            rc = make_map(&map_b, B, b_rows_mem, p.K, ldb, 128);
            if (rc == CF_OK) rc = make_map(&map_a, A, p.M, p.K, lda, tn);
            if (rc != CF_OK) return rc;
            if (tn == 16) return launch_narrow_any<16>(map_b, map_a, p, splits, b_per, st);
            if (tn == 32) return launch_narrow_any<32>(map_b, map_a, p, splits, b_per, st);
            return launch_narrow_any<64>(map_b, map_a, p, splits, b_per, st);
        }
    }
    rc = p.a_mn ? make_map(&map_a, A, p.K, p.M, lda, BK) : make_map(&map_a, A, p.M, p.K, lda, BM);
    if (rc == CF_OK) rc = p.b_mn ? make_map(&map_b, B, b_rows_mem, p.N, ldb, BK) : make_map(&map_b, B, b_rows_mem, p.K, ldb, pair ? 128 : 256);
    if (rc != CF_OK) return rc;
    const bool f32 = p.out_kind == OUT_F32 || p.out_kind == OUT_F32_ADD;
    p.tma_out = p.out_kind != OUT_BF16_ADD && aligned(p.C, 16) && p.ldc % (f32 ? 4 : 8) == 0 && p.N >= (f32 ? 32 : 64);
    if (p.tma_out) {
        rc = f32 ? make_map_c_f32(&map_c, p.C, p.M, p.N, p.ldc) : make_map_c(&map_c, p.C, p.M, p.N, p.ldc);
        if (rc != CF_OK) return rc;
    } else {
        map_c = map_a;                      // not read by the kernel
    }
    // Bands of 8 row blocks keep the slabs of the tiles in flight smallest; a B operand larger than L2 is streamed from HBM once
    // per band, and a taller band pays as long as its own rows of A stay within about 32 MB (the rule and the measurements of
    // the per-tensor GEMM; over seconds, 16384 x 28672 x 4096: 2.05 / 2.02 / 2.00 ms with 8 / 16 / 32).
    if (p.groups == 0 && !p.a_mn && static_cast<long long>(p.N) * p.K > (64ll << 20)) p.raster_m = p.K <= 4096 ? 32 : p.K <= 8192 ? 16 : 8;
    const int tm = pair ? 256 : 128;
    const long long tiles = (cdiv(p.M, tm) + p.groups) * cdiv(p.N, BN);
    if (tiles > 0x3fffffffll) { set_error("%s: product too large", fn); return CF_ERR_LIMIT; }
    const long long most = pair ? pairs : sm_count();
    const int units = static_cast<int>(tiles < most ? tiles : most);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(pair ? 2 * units : units);
    cfg.blockDim = dim3(NUM_THREADS);
    cfg.dynamicSmemBytes = pair ? Cfg<true>::SMEM_BYTES : Cfg<false>::SMEM_BYTES;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = 2; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = pair ? 2 : 1;
    if (pair && b_per == 1) CF_CUDA(cudaLaunchKernelEx(&cfg, k_gemm_b128<true, true>, map_a, map_b, map_c, p));
    else if (pair) CF_CUDA(cudaLaunchKernelEx(&cfg, k_gemm_b128<true, false>, map_a, map_b, map_c, p));
    else if (b_per == 1) CF_CUDA(cudaLaunchKernelEx(&cfg, k_gemm_b128<false, true>, map_a, map_b, map_c, p));
    else CF_CUDA(cudaLaunchKernelEx(&cfg, k_gemm_b128<false, false>, map_a, map_b, map_c, p));
    CF_LAUNCH_CHECK("gemm_b128");
    return CF_OK;
}

int out_kind(int out_fp32, int accumulate) {
    return out_fp32 ? (accumulate ? OUT_F32_ADD : OUT_F32) : (accumulate ? OUT_BF16_ADD : OUT_BF16);
}

// What every form checks. Rows of A: M x K (or K x M), of B: N x K (or K x N).
int check_common(const char* fn, cf_ctx* ctx, int M, int N, int K, const void* A, const void* sa, const void* B, const void* sb,
                 const void* C, long long ldc, int fp32) {
    CF_REQUIRE(ctx != nullptr, "%s: null context", fn);
    CF_REQUIRE(M >= 0 && N >= 0 && K >= 0, "%s: negative shape", fn);
    if (M == 0 || N == 0) return CF_OK;
    constexpr int kMost = 0x7ffffc00;       // tile coordinates are 32-bit
    if (M > kMost || N > kMost || K > kMost) { set_error("%s: a size beyond 2^31 - 1024", fn); return CF_ERR_LIMIT; }
    CF_REQUIRE(C, "%s: null output", fn);
    CF_REQUIRE(ldc >= N, "%s: output pitch smaller than a row", fn);
    CF_REQUIRE(aligned(C, fp32 ? 4 : 2), "%s: misaligned pointer", fn);
    if (K == 0) return CF_OK;
    CF_REQUIRE(A && B, "%s: null matrix pointer", fn);
    CF_REQUIRE(sa && sb, "%s: null descale pointer", fn);
    CF_REQUIRE(aligned(sa, 4) && aligned(sb, 4), "%s: misaligned pointer", fn);
    return CF_OK;
}
// A sum over nothing (K = 0): zero, or what was there.
int empty_contraction(void* C, long long ldc, int M, int N, int fp32, int accumulate, cudaStream_t st) {
    const size_t es = fp32 ? 4 : 2;
    if (!accumulate) CF_CUDA(cudaMemset2DAsync(C, ldc * es, 0, N * es, M, st));
    return CF_OK;
}

}  // namespace
}  // namespace cf

using namespace cf;

extern "C" {

int cf_gemm_fp8_block128_nt(cf_ctx* ctx, int M, int N, int K, const void* d_A, int lda, int a_is_e5m2, const float* d_a_descale,
                            long long a_descale_ld_row, long long a_descale_ld_block, const void* d_B, int ldb, const float* d_b_descale,
                            long long b_descale_ld_row, long long b_descale_ld_block, int b_rows_per_scale, void* d_C, int ldc,
                            int out_fp32, int accumulate, void* stream) {
    const char* fn = "cf_gemm_fp8_block128_nt";
    const int rc = check_common(fn, ctx, M, N, K, d_A, d_a_descale, d_B, d_b_descale, d_C, ldc, out_fp32);
    if (rc != CF_OK || M == 0 || N == 0) return rc;
    if (K == 0) return empty_contraction(d_C, ldc, M, N, out_fp32, accumulate, as_stream(stream));
    CF_REQUIRE(lda >= K && ldb >= K, "%s: operand pitch smaller than a row", fn);
    CF_REQUIRE(b_rows_per_scale == 128 || b_rows_per_scale == 1, "%s: a scale of B covers 128 rows or 1", fn);
    Params p;
    p.M = M; p.N = N; p.K = K;
    p.sa = d_a_descale; p.sa_row = a_descale_ld_row; p.sa_blk = a_descale_ld_block;
    p.sb = d_b_descale; p.sb_row = b_descale_ld_row; p.sb_blk = b_descale_ld_block;
    p.C = d_C; p.ldc = ldc; p.out_kind = out_kind(out_fp32, accumulate);
    p.a_e5m2 = a_is_e5m2 ? 1 : 0;
    return launch_b128(fn, ctx, d_A, lda, d_B, ldb, N, p, b_rows_per_scale, as_stream(stream));
}

int cf_gemm_fp8_block128_nt_grouped(cf_ctx* ctx, int num_experts, int max_total_rows, int N, int K, const int* d_counts,
                                    const int* d_offsets, const void* d_A, int lda, int a_is_e5m2, const float* d_a_descale,
                                    long long a_descale_ld_row, long long a_descale_ld_block, const void* d_B, int ldb,
                                    const float* d_b_descale, long long b_descale_ld_row, long long b_descale_stride, void* d_C, int ldc,
                                    void* stream) {
    const char* fn = "cf_gemm_fp8_block128_nt_grouped";
    const int rc = check_common(fn, ctx, max_total_rows, N, K, d_A, d_a_descale, d_B, d_b_descale, d_C, ldc, 0);
    if (rc != CF_OK || max_total_rows == 0 || N == 0) return rc;
    CF_REQUIRE(K > 0, "%s: empty contraction", fn);
    CF_REQUIRE(num_experts > 0 && d_counts && d_offsets, "%s: no groups", fn);
    if (num_experts > 65536) { set_error("%s: more than 65536 experts", fn); return CF_ERR_LIMIT; }
    CF_REQUIRE(aligned(d_counts, 4) && aligned(d_offsets, 4), "%s: misaligned pointer", fn);
    CF_REQUIRE(lda >= K && ldb >= K, "%s: operand pitch smaller than a row", fn);
    if (static_cast<long long>(num_experts) * N > 0x7fffffffll) { set_error("%s: more than 2^31 weight rows", fn); return CF_ERR_LIMIT; }
    Params p;
    p.M = max_total_rows; p.N = N; p.K = K;
    p.groups = num_experts; p.d_counts = d_counts; p.d_offsets = d_offsets;
    p.sa = d_a_descale; p.sa_row = a_descale_ld_row; p.sa_blk = a_descale_ld_block;
    p.sb = d_b_descale; p.sb_row = b_descale_ld_row; p.sb_blk = 1; p.sb_group = b_descale_stride;
    p.C = d_C; p.ldc = ldc; p.out_kind = OUT_BF16;
    p.a_e5m2 = a_is_e5m2 ? 1 : 0;
    return launch_b128(fn, ctx, d_A, lda, d_B, ldb, static_cast<long long>(num_experts) * N, p, 128, as_stream(stream));
}

int cf_gemm_fp8_block128_nn(cf_ctx* ctx, int M, int N, int K, const void* d_A, int lda, int a_is_e5m2, const float* d_a_descale,
                            long long a_descale_ld_row, long long a_descale_ld_block, const void* d_B_kn, int ldb,
                            const float* d_b_descale, long long b_descale_ld_row, void* d_C, int ldc, int out_fp32, int accumulate,
                            void* stream) {
    const char* fn = "cf_gemm_fp8_block128_nn";
    const int rc = check_common(fn, ctx, M, N, K, d_A, d_a_descale, d_B_kn, d_b_descale, d_C, ldc, out_fp32);
    if (rc != CF_OK || M == 0 || N == 0) return rc;
    if (K == 0) return empty_contraction(d_C, ldc, M, N, out_fp32, accumulate, as_stream(stream));
    CF_REQUIRE(lda >= K && ldb >= N, "%s: operand pitch smaller than a row", fn);
    Params p;
    p.M = M; p.N = N; p.K = K;
    p.sa = d_a_descale; p.sa_row = a_descale_ld_row; p.sa_blk = a_descale_ld_block;
    p.sb = d_b_descale; p.sb_row = 1; p.sb_blk = b_descale_ld_row;      // scales lie [K / 128, N / 128], like the blocks of B
    p.C = d_C; p.ldc = ldc; p.out_kind = out_kind(out_fp32, accumulate);
    p.a_e5m2 = a_is_e5m2 ? 1 : 0;
    p.b_mn = 1;
    return launch_b128(fn, ctx, d_A, lda, d_B_kn, ldb, K, p, 128, as_stream(stream));
}

int cf_gemm_fp8_block128_dw(cf_ctx* ctx, int M, int N, int K, const void* d_X, int ldx, int x_is_e5m2, const float* d_x_descale,
                            long long x_descale_ld_block, long long x_descale_ld_col, const void* d_dY, int ldy, int dy_is_e5m2,
                            const float* d_dy_descale, long long dy_descale_ld_block, long long dy_descale_ld_col, void* d_dW, int ldc,
                            int out_fp32, int accumulate, void* stream) {
    const char* fn = "cf_gemm_fp8_block128_dw";
    const int rc = check_common(fn, ctx, M, N, K, d_X, d_x_descale, d_dY, d_dy_descale, d_dW, ldc, out_fp32);
    if (rc != CF_OK || M == 0 || N == 0) return rc;
    if (K == 0) return empty_contraction(d_dW, ldc, M, N, out_fp32, accumulate, as_stream(stream));
    CF_REQUIRE(ldx >= M && ldy >= N, "%s: operand pitch smaller than a row", fn);
    Params p;
    p.M = M; p.N = N; p.K = K;
    p.sa = d_x_descale; p.sa_row = x_descale_ld_col; p.sa_blk = x_descale_ld_block;
    p.sb = d_dy_descale; p.sb_row = dy_descale_ld_col; p.sb_blk = dy_descale_ld_block;
    p.C = d_dW; p.ldc = ldc; p.out_kind = out_kind(out_fp32, accumulate);
    p.a_e5m2 = x_is_e5m2 ? 1 : 0;
    p.b_e5m2 = dy_is_e5m2 ? 1 : 0;
    p.a_mn = p.b_mn = 1;
    return launch_b128(fn, ctx, d_X, ldx, d_dY, ldy, K, p, 1, as_stream(stream));
}

}  // extern "C"
