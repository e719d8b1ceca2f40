// Product of two microscaled 4-bit matrices, Y[M,N] = A[M,K] * W[N,K]^T, with the per-token and per-channel factors and
// the bias in the epilogue. No counterpart in the reference.
//
// The tensor cores take the format as it is: tcgen05.mma with block scaling multiplies packed e2m1 operands from shared
// memory (64 columns of K per instruction) and takes each block's scale from TMEM. A stage of either kernel is 256 columns
// of K: 128-byte rows of codes (128-byte swizzle) and the scale tiles that go with them, all brought by TMA; tcgen05.cp
// then spreads each 512-byte scale tile (128 rows x 4 blocks) over four TMEM columns. Copies and MMAs are issued by one
// thread and execute in its order, so one set of TMEM columns for the scales serves all stages.
//
//   fp4_pair_kernel   many tokens: CTA pairs, 256 tokens x 256 (128) channels per tile, one persistent pair per two SMs
//   fp4_swap_kernel   few tokens: the weights are the 128-row operand and the tokens (16 .. 128) the MMA's N, so that a
//                     decode step streams weights and wastes no MMA on absent tokens; K is split over a cluster
#include <cuda.h>

#include <type_traits>

#include "fp4_common.cuh"
#include "gemm_tc_shared.cuh"
#include "trace_range.h"

namespace duq4 {

__device__ int g_fp4_status = 0;

int fp4_quantize_rows(int format, int dtype, const void *x, uint32_t rows, uint32_t cols, uint64_t ldx, uint8_t *codes, uint8_t *block_scales,
                      float *row_scales, cudaStream_t st);

extern std::atomic<int> g_static_weights;   // duq4_set_static_weights

namespace fp4 {

using namespace ptx;
using namespace tc;

struct GemmArgs {
    uint32_t M, N, K;
    const uint8_t *a, *a_scales, *w, *w_scales;
    const float *a_rows, *w_rows;   // factor per token / per channel, or null
    const void *bias;
    void *out;
    uint64_t ldo;
};

constexpr int kBK = 256;            // K per stage: 128 bytes of codes per row
constexpr int kTileBytes = 512;     // scale tile: 128 rows x 4 blocks

// Bounded wait on a barrier of this CTA (arrivals may come from the partner).
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile int *abort_flag, int code) {
    return mbar_wait(bar, parity, abort_flag, &g_fp4_status, code);
}
// The wait itself, run out: one warp waits on a barrier that nothing arrives at. `gave_up`: 1 if the first wait reported so, 2 more
// if the next one, with the CTA aborting, did not wait again.
__global__ void fp4_wait_selftest_kernel(int *gave_up) {
    __shared__ int abort_flag;
    __shared__ __align__(8) uint64_t bar;
    if (threadIdx.x == 0) {
        abort_flag = 0;
        mbar_init(smem_u32(&bar), 1);
    }
    __syncthreads();
    const bool first = wait(smem_u32(&bar), 0, &abort_flag, 14);
    const uint64_t t0 = globaltimer();
    const bool second = wait(smem_u32(&bar), 0, &abort_flag, 15);
    if (threadIdx.x == 0) *gave_up = (first ? 0 : 1) + (!second && globaltimer() - t0 < kPtxWaitLimitNs / 2 ? 2 : 0);
}

// Instruction descriptor of the block-scaled kinds: e2m1 x e2m1 -> f32, both operands K-major. (Bits 4-5 and 29-30 name the
// bytes of the 32-bit scale words that an instruction takes: 0 or 2; two scales per instruction of the 32-blocks, four of
// the 16-blocks.)
template <int FMT>
__device__ __forceinline__ uint32_t block_idesc(int m, uint32_t n) {
    return (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((FMT == kMX ? 1u : 0u) << 23) | ((uint32_t)(m >> 4) << 24);
}
// Scale tile in shared memory for tcgen05.cp: 8 rows of 16 bytes are contiguous, groups of 8 rows 128 bytes apart.
__device__ __forceinline__ uint64_t scale_desc(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)1 << 16 | (uint64_t)(128u >> 4) << 32 | (uint64_t)1 << 46;
}
template <int CG>
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint64_t desc) {
    if (CG == 2) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
    else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
#define DUQ4_FP4_MMA(GROUP, KIND)                                                                                          \
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"                                                           \
                 "tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], %1, %2, %3, [%4], [%5], p;\n\t}"                     \
                 ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory")
template <int FMT, int CG>
__device__ __forceinline__ void mma(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    if (FMT == kMX && CG == 2) DUQ4_FP4_MMA("2", "mxf4.block_scale.scale_vec::2X");
    if (FMT == kMX && CG == 1) DUQ4_FP4_MMA("1", "mxf4.block_scale.scale_vec::2X");
    if (FMT == kNV && CG == 2) DUQ4_FP4_MMA("2", "mxf4nvf4.block_scale.scale_vec::4X");
    if (FMT == kNV && CG == 1) DUQ4_FP4_MMA("1", "mxf4nvf4.block_scale.scale_vec::4X");
}
#undef DUQ4_FP4_MMA

// One thread of a warp that runs converged: the operands of what it issues then stay in uniform registers. A stage takes
// up to 18 issues; with the loop on one lane alone each took about 50 ns (4096 x 8192 x 28672, nvfp4: 0.83 ms).
__device__ __forceinline__ bool elected() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
// One stage: its scale tiles to TMEM, its four MMAs. Scale tiles lie [block of 128 rows][tile] in shared memory and
// [tile][block of rows] in TMEM (four columns each), so that the rows of one MMA are contiguous. BB: 128-row blocks of B.
template <int FMT, int CG, int BB>
__device__ __forceinline__ void issue_stage(uint32_t d, uint64_t da, uint64_t db, uint64_t dsa, uint64_t dsb, uint32_t ta, uint32_t tb, uint32_t idesc0,
                                            bool first) {
    constexpr int kTiles = kBK / (4 * (int)block_of(FMT));   // 2 or 4 scale tiles per stage and block of rows
#pragma unroll
    for (int j = 0; j < kTiles; ++j) copy_scales<CG>(ta + j * 4, dsa + j * (kTileBytes >> 4));
#pragma unroll
    for (int j = 0; j < kTiles; ++j)
#pragma unroll
        for (int b = 0; b < BB; ++b) copy_scales<CG>(tb + (j * BB + b) * 4, dsb + (b * kTiles + j) * (kTileBytes >> 4));
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
        const int j = FMT == kMX ? kk >> 1 : kk;
        const uint32_t sf = FMT == kMX ? (kk & 1) * 2 : 0;
        mma<FMT, CG>(d, da + (uint64_t)(kk * 2), db + (uint64_t)(kk * 2), idesc0 | (sf << 4) | (sf << 29), ta + j * 4, tb + j * BB * 4, !first || kk > 0);
    }
}

// y = acc * channel factor * token factor + bias. The channel's first: weights are about as large in every layer, while tokens reach
// over the range of bfloat16, and a sum of up to 2^23 K times the token's factor alone would leave that of 32 bits.
__device__ __forceinline__ float finish(float acc, float ra, float rw, float b) { return __fmaf_rn(__fmul_rn(acc, rw), ra, b); }

__device__ __forceinline__ uint32_t ctarank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t in_cta(uint32_t local_addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local_addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void arrive_at(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
template <int CG>
__device__ __forceinline__ void commit(uint32_t cluster_bar) {
    if (CG == 2) asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(cluster_bar) : "memory");
    else asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(cluster_bar) : "memory");
}
// Copies whose bytes are credited to a barrier of either CTA of the pair (CG == 2) or of this CTA.
template <int CG>
__device__ __forceinline__ void load_2d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y) {
    if (CG == 2)
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
                     "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst), "l"(map),
                     "r"(bar), "r"(x), "r"(y) : "memory");
}
template <int CG>
__device__ __forceinline__ void load_3d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z) {
    if (CG == 2)
        asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
                     "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
    else
        tma_load_3d(dst, map, bar, x, y, z);
}

// ---- many tokens: CTA pairs -------------------------------------------------------------------------------------
struct PairArgs {
    GemmArgs g;
    uint32_t tiles_m, tiles_n, bn;   // tiles of 256 tokens x bn channels (128 or 256)
};

template <int FMT>
struct Pair {
    static constexpr int kTiles = kBK / (4 * (int)block_of(FMT));
    static constexpr int kStages = FMT == kMX ? 6 : 5;
    static constexpr int kOperand = 128 * 128;                 // one CTA's 128 rows of codes
    static constexpr int kScaleA = kTiles * kTileBytes, kScaleStage = 3 * kScaleA;   // own tokens, then all channels of the tile
    static constexpr int kStore = 1024;                        // an epilogue warp's 32 rows x 16 channels,
    static constexpr int kTerms = 128 * 6;                     // and the factors (float) and biases (16 bits) of its 128 channels
    static constexpr int kSmem = 1024 + kStages * (2 * kOperand + kScaleStage) + 8 * (kStore + kTerms);
    static constexpr int kThreads = 32 * 10;
    // TMEM: two accumulators of 256 columns and the scales do not fit in 512 columns side by side, so the second
    // accumulator starts inside the first: its first 64 columns are the first one's last 64. The epilogue takes those
    // columns first and lets the next tile start when it has them in registers.
    static constexpr uint32_t kSecond = 192, kSfa = 448, kSfb = 448 + 4 * kTiles;
    static_assert(kSfb + 8 * kTiles <= 512 && kSmem <= 232448 - 512, "does not fit");
};

// A warp's 32 tokens (one per lane) x 32 neighbouring channels from the accumulator to memory. f, bias: the channels'
// factors and biases in shared memory; how: rows of the result start on 32 (2) or 16 (1) bytes or neither (0). `stage`: the
// warp's 1 KiB.
template <class T>
__device__ __forceinline__ void store32(const GemmArgs &a, const uint32_t (&v)[32], uint32_t m0, uint32_t n, float ra, const float *f, const uint32_t *bias,
                                        int how, uint8_t *stage) {
    const int lane = threadIdx.x & 31;
    const uint32_t m = m0 + lane;
    const bool inside = n + 32 <= a.N;
    uint16_t *out = reinterpret_cast<uint16_t *>(a.out);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t o[8];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float4 fq = *reinterpret_cast<const float4 *>(f + h * 16 + q * 4);
            const uint2 bq = *reinterpret_cast<const uint2 *>(bias + h * 8 + q * 2);
            const float2 b0 = Two<T>::up(bq.x), b1 = Two<T>::up(bq.y);
            const int e = h * 16 + q * 4;
            o[2 * q] = Two<T>::down(finish(__uint_as_float(v[e]), ra, fq.x, b0.x), finish(__uint_as_float(v[e + 1]), ra, fq.y, b0.y));
            o[2 * q + 1] = Two<T>::down(finish(__uint_as_float(v[e + 2]), ra, fq.z, b1.x), finish(__uint_as_float(v[e + 3]), ra, fq.w, b1.y));
        }
        if (how && inside) {
            uint16_t *row = out + (size_t)m * a.ldo + n + h * 16;
            if (m < a.M) {
                if (how == 2) {
                    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(row), "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]),
                                 "r"(o[4]), "r"(o[5]), "r"(o[6]), "r"(o[7]) : "memory");
                } else {
                    reinterpret_cast<uint4 *>(row)[0] = make_uint4(o[0], o[1], o[2], o[3]);
                    reinterpret_cast<uint4 *>(row)[1] = make_uint4(o[4], o[5], o[6], o[7]);
                }
            }
        } else {
            // rows of any alignment: through shared memory, so that neighbouring lanes store neighbouring channels
            // (stored lane by lane, 32 segments per instruction, a tile of 256 x 256 took longer than its MMAs)
            reinterpret_cast<uint4 *>(stage + lane * 32)[0] = make_uint4(o[0], o[1], o[2], o[3]);
            reinterpret_cast<uint4 *>(stage + lane * 32)[1] = make_uint4(o[4], o[5], o[6], o[7]);
            __syncwarp();
            const uint32_t c = n + h * 16 + (lane & 15);
#pragma unroll 4
            for (int r = lane >> 4; r < 32; r += 2)
                if (m0 + r < a.M && c < a.N) out[(size_t)(m0 + r) * a.ldo + c] = reinterpret_cast<const uint16_t *>(stage)[r * 16 + (lane & 15)];
            __syncwarp();
        }
    }
}

template <int FMT, class T>
__global__ void __launch_bounds__(Pair<FMT>::kThreads, 1)
fp4_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_sa,
                const __grid_constant__ CUtensorMap map_sw, const PairArgs p) {
    using C = Pair<FMT>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    __shared__ __align__(8) uint64_t bars[2 * C::kStages + 6];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u, scales0 = base + C::kStages * 2 * C::kOperand, bar0 = smem_u32(bars);
    auto full = [&](int s) { return bar0 + 8u * s; };                        // the leader's: both CTAs' copies
    auto empty = [&](int s) { return bar0 + 8u * (C::kStages + s); };        // each CTA's: the MMAs that read the stage
    auto acc_full = [&](int b) { return bar0 + 8u * (2 * C::kStages + b); }; // each CTA's
    auto acc_empty = [&](int b) { return bar0 + 8u * (2 * C::kStages + 2 + b); };   // the leader's: epilogue warps of both
    const uint32_t shared_free = bar0 + 8u * (2 * C::kStages + 4);           // the leader's: the shared columns are read
    const uint32_t drained = bar0 + 8u * (2 * C::kStages + 5);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // uniform
    const uint32_t rank = ctarank(), pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
    const uint32_t tiles = p.tiles_m * p.tiles_n, ksteps = (p.g.K + kBK - 1) / kBK, bn = p.bn;

    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(acc_full(b), 1);
            mbar_init(acc_empty(b), 16);
        }
        mbar_init(shared_free, 16);
        mbar_init(drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_barrier();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    volatile int *abortp = &abort_flag;

    // Tile order: token blocks fastest inside bands of 16, so that the pairs at work share a few weight tiles and a band of
    // activations that stays in L2.
    auto coords = [&](uint32_t t, uint32_t &tm, uint32_t &tn) {
        const uint32_t per_band = 16 * p.tiles_n, band = t / per_band, r = t % per_band, here = min(16u, p.tiles_m - band * 16);
        tn = r / here;
        tm = band * 16 + r % here;
    };

    asm volatile("griddepcontrol.wait;" ::: "memory");   // the launch in front may still have run so far
    // the rest of the columns, where a second launch does them, may start: the tokens are there
    if (threadIdx.x == 0) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (warp == 0) {
        uint32_t s = 0, ph = 0;
        bool ok = true;
        const uint32_t bytes = 2 * (C::kOperand + bn / 2 * 128 + C::kScaleA * (1 + bn / 128));
        for (uint32_t t = pair; ok && t < tiles; t += npairs) {
            uint32_t tm, tn;
            coords(t, tm, tn);
            for (uint32_t ks = 0; ks < ksteps; ++ks) {
                if (!(ok = wait(empty(s), ph ^ 1, abortp, 1))) break;
                if (elected()) {
                    if (rank == 0) mbar_expect_tx(full(s), bytes);
                    const uint32_t bar = in_cta(full(s), 0), dst = base + s * 2 * C::kOperand, sc = scales0 + s * C::kScaleStage;
                    load_2d<2>(dst, &map_a, bar, ks * 128, tm * 256 + rank * 128);
                    load_2d<2>(dst + C::kOperand, &map_w, bar, ks * 128, tn * bn + rank * (bn / 2));
                    load_3d<2>(sc, &map_sa, bar, 0, ks * C::kTiles, tm * 2 + rank);
                    load_3d<2>(sc + C::kScaleA, &map_sw, bar, 0, ks * C::kTiles, tn * (bn / 128));
                }
                __syncwarp();
                if (++s == C::kStages) { s = 0; ph ^= 1; }
            }
        }
        if (!ok) leave_copies_behind();
    } else if (warp == 1) {
        if (rank == 0) {
            uint32_t s = 0, ph = 0, lt = 0;
            bool ok = true, issued = false;
            const bool wide = bn == 256;
            const uint32_t idesc = block_idesc<FMT>(256, bn);
            const uint64_t desc_a = make_desc(base), desc_s = scale_desc(scales0);
            for (uint32_t t = pair; ok && t < tiles; t += npairs, ++lt) {
                const uint32_t buf = lt & 1;
                if (!(ok = wait(acc_empty(buf), ((lt >> 1) & 1) ^ 1, abortp, 2))) break;
                if (lt > 0 && !(ok = wait(shared_free, (lt - 1) & 1, abortp, 3))) break;
                tc_fence_after();
                const uint32_t d = tmem + buf * C::kSecond;
                for (uint32_t ks = 0; ks < ksteps; ++ks) {
                    if (!(ok = wait(full(s), ph, abortp, 4))) break;
                    tc_fence_after();
                    const uint64_t da = desc_a + s * (2 * C::kOperand >> 4), ds = desc_s + s * (C::kScaleStage >> 4);
                    if (elected()) {
                        if (wide)
                            issue_stage<FMT, 2, 2>(d, da, da + (C::kOperand >> 4), ds, ds + (C::kScaleA >> 4), tmem + C::kSfa, tmem + C::kSfb, idesc, ks == 0);
                        else
                            issue_stage<FMT, 2, 1>(d, da, da + (C::kOperand >> 4), ds, ds + (C::kScaleA >> 4), tmem + C::kSfa, tmem + C::kSfb, idesc, ks == 0);
                        commit<2>(empty(s));
                        commit<2>(in_cta(empty(s), 1));
                        if (ks + 1 == ksteps) {
                            commit<2>(acc_full(buf));
                            commit<2>(in_cta(acc_full(buf), 1));
                        }
                    }
                    __syncwarp();
                    issued = true;
                    if (++s == C::kStages) { s = 0; ph ^= 1; }
                }
            }
            if (!ok && issued) {
                if (elected()) commit<2>(drained);
                const uint64_t t0 = globaltimer();
                while (!mbar_try(drained, 0) && globaltimer() - t0 < kPtxWaitLimitNs) __nanosleep(1000);
            }
            if (!ok) leave_copies_behind();   // both producers may have issued their last copies long ago; the pair ends together
        }
    } else {
        // Epilogue, eight warps: two per TMEM lane quadrant, which take the tile's 32-column chunks in turn, the shared
        // ones (6, 7 of the first accumulator, 0, 1 of the second) first.
        const int quad = warp & 3, half = (warp - 2) >> 2;
        const uintptr_t rows = reinterpret_cast<uintptr_t>(p.g.out) | (uintptr_t)(p.g.ldo * 2);
        const int how = (rows & 31) == 0 ? 2 : (rows & 15) == 0 ? 1 : 0;
        uint8_t *stage = smem_raw + (scales0 + C::kStages * C::kScaleStage - smem_u32(smem_raw)) + (warp - 2) * (C::kStore + C::kTerms);
        float *factors = reinterpret_cast<float *>(stage + C::kStore);
        uint16_t *biases = reinterpret_cast<uint16_t *>(factors + 128);
        uint32_t lt = 0;
        for (uint32_t t = pair; t < tiles; t += npairs, ++lt) {
            uint32_t tm, tn;
            coords(t, tm, tn);
            const uint32_t buf = lt & 1, m0 = tm * 256 + rank * 128 + quad * 32, m = m0 + lane;
            const float ra = m < p.g.M && p.g.a_rows ? p.g.a_rows[m] : 1.f;
            // this warp's four chunks' channel terms, fetched while the tile is computed
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t n = tn * bn + ((2 * i + half + (buf ? 0 : 6)) & 7) * 32 + lane;
                const bool in = n < p.g.N;
                factors[i * 32 + lane] = in && p.g.w_rows ? p.g.w_rows[n] : 1.f;
                biases[i * 32 + lane] = in && p.g.bias ? reinterpret_cast<const uint16_t *>(p.g.bias)[n] : (uint16_t)0;
            }
            __syncwarp();
            if (!wait(acc_full(buf), (lt >> 1) & 1, abortp, 5)) break;
            tc_fence_after();
            const uint32_t acc = tmem + buf * C::kSecond + ((uint32_t)(quad * 32) << 16);
#pragma unroll 1
            for (int i = 0; i < 4; ++i) {
                const uint32_t ch = (2 * i + half + (buf ? 0 : 6)) & 7, n = tn * bn + ch * 32;
                uint32_t v[32];
                if (ch * 32 < bn) {
                    __syncwarp();
                    tmem_ld32(acc + ch * 32, v);
                    tmem_ld_wait();
                }
                if (i == 0 || i == 3) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) arrive_at(in_cta(i == 0 ? shared_free : acc_empty(buf), 0));
                }
                if (ch * 32 < bn && m0 < p.g.M && n < p.g.N) store32<T>(p.g, v, m0, n, ra, factors + i * 32, reinterpret_cast<const uint32_t *>(biases + i * 32), how, stage);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_barrier();   // the partner is done with this CTA's shared memory and TMEM
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// ---- few tokens: weights as the 128-row operand ---------------------------------------------------------------
struct SwapArgs {
    GemmArgs g;
    uint32_t nt, splits;     // tokens per tile (a multiple of 16; 128 where there are several tiles); CTAs that share a tile's K
    uint32_t tmem_cols;
    uint32_t stages;
    // What the launch in front, which may still run, leaves this one: 1: the weights are there (it is the tokens' quantizer, or the
    // caller has promised so), 2: all is there, 3: nothing
    uint32_t early;
};

template <int FMT>
struct Swap {
    static constexpr int kTiles = kBK / (4 * (int)block_of(FMT));
    static constexpr int kScale = kTiles * kTileBytes;
    static constexpr int kThreads = 32 * 6;
    static constexpr int kMaxStages = 10;
    static __host__ __device__ uint32_t stage_bytes(uint32_t nt) { return 128 * 128 + nt * 128; }   // multiples of 1024
};

template <int FMT, class T>
__global__ void __launch_bounds__(Swap<FMT>::kThreads)
fp4_swap_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_sa,
                const __grid_constant__ CUtensorMap map_sw, const SwapArgs p) {
    using C = Swap<FMT>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    __shared__ __align__(8) uint64_t bars[2 * C::kMaxStages + 2];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u, stage = C::stage_bytes(p.nt), scales0 = base + p.stages * stage;
    float *part = reinterpret_cast<float *>(smem_raw + (base - smem_u32(smem_raw)));   // [token][128 channels], over the stages
    const uint32_t bar0 = smem_u32(bars);
    auto full = [&](uint32_t s) { return bar0 + 8u * s; };
    auto empty = [&](uint32_t s) { return bar0 + 8u * (C::kMaxStages + s); };
    const uint32_t acc_full = bar0 + 8u * 2 * C::kMaxStages, drained = acc_full + 8;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // uniform
    const uint32_t rank = p.splits > 1 ? ctarank() : 0;
    const uint32_t tn = blockIdx.x / p.splits, t0 = blockIdx.y * p.nt;
    const uint32_t ktiles = (p.g.K + kBK - 1) / kBK, k0 = rank * ktiles / p.splits, k1 = (rank + 1) * ktiles / p.splits;

    const uint32_t head = min(p.stages, k1 - k0);   // the first round of stages
    auto weights = [&](uint32_t k, uint32_t s) {    // a stage's weights, and the bytes it waits for
        mbar_expect_tx(full(s), stage + 2 * C::kScale);
        load_2d<1>(base + s * stage, &map_w, full(s), k * 128, tn * 128);
        load_3d<1>(scales0 + s * 2 * C::kScale, &map_sw, full(s), 0, k * C::kTiles, tn);
    };
    auto tokens = [&](uint32_t k, uint32_t s) {
        load_2d<1>(base + s * stage + 128 * 128, &map_a, full(s), k * 128, t0);
        load_3d<1>(scales0 + s * 2 * C::kScale + C::kScale, &map_sa, full(s), 0, k * C::kTiles, t0 >> 7);
    };
    if (warp == 0) {
        if (elected()) {
            abort_flag = 0;
            for (uint32_t s = 0; s < p.stages; ++s) {
                mbar_init(full(s), 1);
                mbar_init(empty(s), 1);
            }
            mbar_init(acc_full, 1);
            mbar_init(drained, 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            fence_proxy_async();   // the copies find the barriers initialised
        }
        __syncwarp();
        asm volatile("bar.arrive 1, %0;" ::"n"(C::kThreads) : "memory");   // the barriers are there; nothing of the others is needed
        if (p.early == 3) asm volatile("griddepcontrol.wait;" ::: "memory");
        for (uint32_t i = 0; i < head; ++i) {
            if (elected()) {
                weights(k0 + i, i);
                if (p.early != 1) tokens(k0 + i, i);
            }
            __syncwarp();
        }
    } else {
        if (warp == 1) {
            tmem_alloc(smem_u32(&tmem_slot), p.tmem_cols);
            tmem_relinquish();
            // the next launch on the stream may set itself up (and take TMEM: not before this one has its own); it waits for this one
            asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
        }
        tc_fence_before();
        asm volatile("bar.sync 1, %0;" ::"n"(C::kThreads) : "memory");
        tc_fence_after();
        if (p.early == 3) asm volatile("griddepcontrol.wait;" ::: "memory");
    }
    const uint32_t tmem = warp == 0 ? 0 : tmem_slot, sfa = tmem + p.nt, sfb = sfa + 4 * C::kTiles;   // columns behind the accumulator
    volatile int *abortp = &abort_flag;

    // what the thread stores: four channels of every so many tokens, and their terms, fetched while the sums are made
    const uint32_t tokens_here = min(p.nt, p.g.M - t0), c = (threadIdx.x & 31) * 4, n = tn * 128 + c;
    uint16_t *out = reinterpret_cast<uint16_t *>(p.g.out);
    const uint16_t *bias = reinterpret_cast<const uint16_t *>(p.g.bias);
    const bool vec = (p.g.ldo & 3) == 0 && (reinterpret_cast<uintptr_t>(out) & 7) == 0 && n + 4 <= p.g.N;
    float f[4], b[4];
    auto terms = [&] {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool in = n + j < p.g.N;
            // plain loads: read-only-path ones may be moved ahead of a wait
            f[j] = in && p.g.w_rows ? p.g.w_rows[n + j] : 1.f;
            b[j] = in && bias ? Two<T>::up1(bias[n + j]) : 0.f;
        }
    };
    if (warp == 0) {
        bool ok = true;
        if (p.early == 1) {
            asm volatile("griddepcontrol.wait;" ::: "memory");
            for (uint32_t i = 0; i < head; ++i) {
                if (elected()) tokens(k0 + i, i);
                __syncwarp();
            }
        }
        uint32_t s = 0, ph = 1;
        for (uint32_t i = head; i < k1 - k0; ++i) {
            if (!(ok = wait(empty(s), ph ^ 1, abortp, 11))) break;
            if (elected()) {
                weights(k0 + i, s);
                tokens(k0 + i, s);
            }
            __syncwarp();
            if (++s == p.stages) { s = 0; ph ^= 1; }
        }
        if (!ok) leave_copies_behind();
    } else if (warp == 1) {
        if (p.early == 1) asm volatile("griddepcontrol.wait;" ::: "memory");   // the launch in front may take longer than a wait on a barrier may
        bool ok = true, issued = false;
        const uint32_t idesc = block_idesc<FMT>(128, p.nt);
        const uint64_t desc_w = make_desc(base), desc_s = scale_desc(scales0);
        uint32_t s = 0, ph = 0;
        for (uint32_t i = 0; i < k1 - k0; ++i) {
            if (!(ok = wait(full(s), ph, abortp, 12))) break;
            tc_fence_after();
            const uint64_t dw = desc_w + s * (stage >> 4), ds = desc_s + s * (2 * C::kScale >> 4);
            if (elected()) {
                issue_stage<FMT, 1, 1>(tmem, dw, dw + (128 * 128 >> 4), ds, ds + (C::kScale >> 4), sfa, sfb, idesc, i == 0);
                commit<1>(empty(s));
                if (i + 1 == k1 - k0) commit<1>(acc_full);
            }
            __syncwarp();
            issued = true;
            if (++s == p.stages) { s = 0; ph ^= 1; }
        }
        if (!ok && issued) {
            if (elected()) commit<1>(drained);
            const uint64_t b0 = globaltimer();
            while (!mbar_try(drained, 0) && globaltimer() - b0 < kPtxWaitLimitNs) __nanosleep(1000);
        }
        if (!ok) leave_copies_behind();   // the producer may have issued its last copy long ago
    } else {
        terms();
        if (p.early == 1) asm volatile("griddepcontrol.wait;" ::: "memory");
        wait(acc_full, 0, abortp, 13);
        tc_fence_after();
    }
    if (warp < 2) terms();
    // From here on the tokens' factors are read and the result is written: unless all is there from the start, every warp has
    // waited for the launch in front.
    if (warp >= 2 && !abort_flag) {
        const uint32_t quad = warp & 3, acc = tmem + ((quad * 32) << 16);
        for (uint32_t c = 0; c < p.nt; c += 16) {
            uint32_t v[16];
            __syncwarp();
            tmem_ld16(acc + c, v);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) part[(c + j) * 128 + quad * 32 + lane] = __uint_as_float(v[j]);
        }
        tc_fence_before();
    }
    // The partial sums of the cluster's CTAs meet in distributed shared memory; each CTA adds and stores a share of the
    // tokens, a token per warp and step and four channels per thread, always in the order of the CTAs. (Sent to the storing
    // CTA instead, 128 tokens, 4096 x 4096: 10.6 us against 9.4; 16 tokens: 6.8 against 7.2.)
    if (p.splits > 1) cluster_barrier();
    else __syncthreads();
    if (warp == 1) {   // the accumulators have been read
        tc_fence_after();
        tmem_dealloc(tmem, p.tmem_cols);
    }
    auto store = [&](uint32_t t, const float4 &y) {
        const uint32_t m = t0 + t;
        const float ra = p.g.a_rows ? p.g.a_rows[m] : 1.f;
        const uint2 w = make_uint2(Two<T>::down(finish(y.x, ra, f[0], b[0]), finish(y.y, ra, f[1], b[1])),
                                   Two<T>::down(finish(y.z, ra, f[2], b[2]), finish(y.w, ra, f[3], b[3])));
        uint16_t *o = out + (size_t)m * p.g.ldo + n;
        if (vec) {
            *reinterpret_cast<uint2 *>(o) = w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n + j < p.g.N) o[j] = (uint16_t)((j < 2 ? w.x : w.y) >> (16 * (j & 1)));
        }
    };
    // U tokens at a time, so that their reads are on the way together
    const uint32_t first = rank * (C::kThreads / 32) + warp, step = p.splits * (C::kThreads / 32);
    auto gather = [&](auto us, auto splits) {
        constexpr int U = decltype(us)::value, S = decltype(splits)::value;
        for (uint32_t t = first; t < tokens_here; t += U * step) {
            float4 v[U][S];
#pragma unroll
            for (int i = 0; i < U; ++i)
#pragma unroll
                for (int s = 0; s < S; ++s)
                    if (t + i * step < tokens_here)
                        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                     : "=f"(v[i][s].x), "=f"(v[i][s].y), "=f"(v[i][s].z), "=f"(v[i][s].w)
                                     : "r"(in_cta(smem_u32(part + (t + i * step) * 128 + c), s)));
#pragma unroll
            for (int i = 0; i < U; ++i) {
                if (t + i * step >= tokens_here) break;
                float4 y = v[i][0];
#pragma unroll
                for (int s = 1; s < S; ++s) { y.x += v[i][s].x; y.y += v[i][s].y; y.z += v[i][s].z; y.w += v[i][s].w; }
                store(t + i * step, y);
            }
        }
    };
    if (!abort_flag && n < p.g.N) {
        using std::integral_constant;
        if (p.splits == 1) {
            for (uint32_t t = first; t < tokens_here; t += step) store(t, *reinterpret_cast<const float4 *>(part + t * 128 + c));
        } else if (p.splits == 2) {
            gather(integral_constant<int, 4>{}, integral_constant<int, 2>{});
        } else if (p.splits == 4) {
            gather(integral_constant<int, 3>{}, integral_constant<int, 4>{});
        } else {
            gather(integral_constant<int, 1>{}, integral_constant<int, 8>{});
        }
    }
    __syncwarp();
    if (p.splits > 1) cluster_barrier();   // the others have read this CTA's partial sums
    if (p.early == 2) asm volatile("griddepcontrol.wait;" ::: "memory");   // this launch does not end before the one in front
}

// ---- launches --------------------------------------------------------------------------------------------------
using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                              const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeFn encoder() {
    static const EncodeFn fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess;
        return ok ? (EncodeFn)p : (EncodeFn) nullptr;
    }();
    return fn;
}
// Codes [rows, K/2] in boxes of 128 bytes x box_rows, 128-byte swizzle. A new descriptor per call: nothing is kept.
static int map_codes(CUtensorMap *m, const uint8_t *p, uint32_t rows, uint32_t K, uint32_t box_rows) {
    const EncodeFn f = encoder();
    if (!f) return DUQ4_ERR_DEVICE;
    const cuuint64_t dims[2] = {K / 2, rows}, strides[1] = {K / 2};
    const cuuint32_t box[2] = {128, box_rows}, one[2] = {1, 1};
    return f(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t *>(p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? DUQ4_OK : DUQ4_ERR_SHAPE;
}
// Block scales as [blocks of 128 rows][tiles of a row][512 bytes]; tiles beyond the row's end read as zero.
static int map_scales(CUtensorMap *m, const uint8_t *p, int format, uint32_t rows, uint32_t K, uint32_t box_blocks) {
    const EncodeFn f = encoder();
    if (!f) return DUQ4_ERR_DEVICE;
    const uint32_t tiles = scale_tiles(format, K), per_stage = kBK / (4 * block_of(format));
    const cuuint64_t dims[3] = {kTileBytes / 4, tiles, cdiv(rows, 128)}, strides[2] = {kTileBytes, (cuuint64_t)tiles * kTileBytes};
    const cuuint32_t box[3] = {kTileBytes / 4, per_stage, box_blocks}, one[3] = {1, 1, 1};
    return f(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, const_cast<uint8_t *>(p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? DUQ4_OK : DUQ4_ERR_SHAPE;
}

template <class F>
static int launch(F *kernel, uint32_t gx, uint32_t gy, uint32_t threads, uint32_t smem, uint32_t cluster, cudaStream_t st, const CUtensorMap (&maps)[4],
                  const void *args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(gx, gy);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    void *a[] = {(void *)&maps[0], (void *)&maps[1], (void *)&maps[2], (void *)&maps[3], const_cast<void *>(args)};
    const cudaError_t e = cudaLaunchKernelExC(&cfg, (const void *)kernel, a);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return (int)e;
    }
    return launch_status();
}

template <int FMT, class T>
static int launch_pair(const GemmArgs &g, cudaStream_t st) {
    using C = Pair<FMT>;
    static DeviceOnce once;
    const int dev = current_device_slot();
    if (dev < 0) return DUQ4_ERR_DEVICE;
    int rc = once.run(dev, [] { return (int)cudaFuncSetAttribute(fp4_pair_kernel<FMT, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem); });
    if (rc) return rc;
    const uint32_t pairs = (uint32_t)sm_count_current_device() / 2;
    PairArgs p{g, cdiv(g.M, 256), 0, 256};
    if ((uint64_t)p.tiles_m * cdiv(g.N, 256) * 2 <= pairs) p.bn = 128;
    p.tiles_n = cdiv(g.N, p.bn);
    CUtensorMap maps[4];
    if ((rc = map_codes(&maps[0], g.a, g.M, g.K, 128)) || (rc = map_codes(&maps[1], g.w, g.N, g.K, p.bn / 2)) ||
        (rc = map_scales(&maps[2], g.a_scales, FMT, g.M, g.K, 1)) || (rc = map_scales(&maps[3], g.w_scales, FMT, g.N, g.K, p.bn / 128)))
        return rc;
    if ((uint64_t)p.tiles_m * p.tiles_n > 0x7FFFFFFFull) return DUQ4_ERR_SHAPE;
    const uint32_t n = p.tiles_m * p.tiles_n < pairs ? p.tiles_m * p.tiles_n : pairs;
    return launch(fp4_pair_kernel<FMT, T>, 2 * n, 1, C::kThreads, C::kSmem, 2, st, maps, &p);
}

// CTAs that share a tile's K: up to eight while there is an SM for each (nvfp4, us with 1 / 2 / 4 / 8: 16 tokens, 4096 x 4096 6.5 /
// 5.7 / 5.5 / 6.3; 1024 x 11008 12.0 / 8.1 / 5.7 / 5.3; 22016 x 4096, 172 tiles: 12.2 / 14.8, whose 344 CTAs do not fit at once).
// With more than 64 tokens the partial sums weigh more: beyond two CTAs, each keeps a step of K for every four tiles (128 tokens:
// 4096 x 4096, 32 tiles, 10.2 / 8.4 / 9.4; 2048 x 2048, 16 tiles, 7.8 / 6.8 / 7.0 / 7.4; 2048 x 11008 16.6 / 11.5 / 10.9 / 10.3).
static uint32_t swap_splits(uint32_t M, uint64_t tiles, uint64_t ktiles, uint64_t sms) {
    uint32_t splits = 1;
    while (splits < 8 && tiles * splits * 2 <= sms && ktiles >= splits * 2 && (M <= 64 || splits == 1 || ktiles * 4 >= splits * 2 * tiles)) splits *= 2;
    return splits;
}
template <int FMT, class T>
static int launch_swap(const GemmArgs &g, cudaStream_t st, uint32_t early) {
    using C = Swap<FMT>;
    constexpr uint32_t kMaxSmem = 232448 - 1024;
    static DeviceOnce once;
    const int dev = current_device_slot();
    if (dev < 0) return DUQ4_ERR_DEVICE;
    int rc = once.run(dev, [] { return (int)cudaFuncSetAttribute(fp4_swap_kernel<FMT, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem); });
    if (rc) return rc;
    SwapArgs p{g, 0, 1, 0, 0, early};
    p.nt = g.M > 128 ? 128 : (g.M + 15) / 16 * 16;
    const uint32_t tiles_n = cdiv(g.N, 128), tiles_m = cdiv(g.M, p.nt), ktiles = cdiv(g.K, (uint32_t)kBK);
    const uint32_t cols = p.nt + 8 * C::kTiles;
    p.tmem_cols = cols <= 64 ? 64 : cols <= 128 ? 128 : 256;
    const uint32_t per_stage = C::stage_bytes(p.nt) + 2 * C::kScale;
    const uint32_t sms = (uint32_t)sm_count_current_device();
    p.splits = swap_splits(g.M, (uint64_t)tiles_n * tiles_m, ktiles, sms);
    // stages: an SM's shared memory for one CTA, or half of it (228 KiB, 1 KiB a CTA taken) for two
    const bool alone = p.splits <= 2 && (uint64_t)tiles_n * tiles_m * p.splits <= sms;   // (wider clusters pack badly one CTA to an SM)
    p.stages = ((alone ? 220 : 111) * 1024) / per_stage;
    if (p.stages > (uint32_t)C::kMaxStages) p.stages = C::kMaxStages;
    if (p.stages > cdiv(ktiles, p.splits)) p.stages = cdiv(ktiles, p.splits);
    uint32_t smem = p.stages * per_stage;
    if (smem < p.nt * 512u) smem = p.nt * 512u;
    smem += 1024;
    // A CTA takes at least as large a part of the SM's shared memory as of its TMEM (64 columns count for a ninth of 228 KiB), so
    // that CTAs whose columns do not fit together are never on one SM together: one that waited there for columns would keep
    // its cluster waiting, and the cluster what others wait for.
    if (smem < p.tmem_cols * 408u) smem = p.tmem_cols * 408u;
    CUtensorMap maps[4];
    if ((rc = map_codes(&maps[0], g.a, g.M, g.K, p.nt)) || (rc = map_codes(&maps[1], g.w, g.N, g.K, 128)) ||
        (rc = map_scales(&maps[2], g.a_scales, FMT, g.M, g.K, 1)) || (rc = map_scales(&maps[3], g.w_scales, FMT, g.N, g.K, 1)))
        return rc;
    return launch(fp4_swap_kernel<FMT, T>, tiles_n * p.splits, tiles_m, C::kThreads, smem, p.splits, st, maps, &p);
}

// Which kernel. Both are priced by the columns of K that the busiest SM goes through, in steps of 256, and a fixed part: for the
// pair kernel with tiles of 256 x 256 or, where those leave half of the pairs idle, 256 x 128; for the other one without and with
// a meeting. The numbers are relative: fitted to both kernels' times at 234 sizes (144 .. 2048 tokens, 1024 .. 28672 channels, K
// 2048 .. 11008, both formats) so that the cheapest is the fastest; in the fit what they choose is at most
// 4 % slower than the best choice. (Measured, nvfp4, pair / swap / whole rounds and rest, us: 256 x 22016 x 4096 18.2 / 25.8 / 21.4; 256 x 4096 x
// 11008 14.9 / 13.1; 300 x 11008 x 4096 16.4 / 14.9 / 19.3; 512 x 4096 x 4096 9.3 / 11.0; 4149 x 45 x 24800 32.7 / 20.7;
// 512 x 28672 x 8192 55.2 / 96.2 / 54.0.)
static uint64_t pair_price(uint64_t tiles, uint64_t ktiles, uint64_t sms) {
    return tiles * 4 <= sms ? ktiles * 50 + 140 : (tiles + sms / 2 - 1) / (sms / 2) * ktiles * 63 + 750;
}
static uint64_t swap_price(uint32_t M, uint64_t tiles, uint64_t ktiles, uint64_t sms) {
    const uint64_t splits = swap_splits(M, tiles, ktiles, sms);
    return (tiles * splits + sms - 1) / sms * ((ktiles + splits - 1) / splits) * 50 + (splits > 1 ? 1120 : 810);
}
// The columns of the result that the pair kernel computes: none, all, or whole rounds of its tiles, the columns that are left
// being the other kernel's (they begin at a multiple of 256, so at a whole tile of the weights' block scales).
static uint32_t pair_columns(uint32_t M, uint32_t N, uint32_t K, uint64_t sms) {
    if (M <= 128) return 0;
    const uint64_t ktiles = cdiv(K, (uint32_t)kBK), tiles_m = cdiv(M, 256), tiles_n = cdiv(N, 256);
    const uint64_t blocks_m = cdiv(M, 128), pairs = pair_price(tiles_m * tiles_n, ktiles, sms);
    const bool swap_fits = blocks_m <= 65535;   // the grid's second dimension
    const uint64_t swap = swap_fits ? swap_price(M, blocks_m * cdiv(N, 128), ktiles, sms) : ~0ull, one = swap < pairs ? swap : pairs;
    // A last round that few tiles are left for: whole rounds by the pair kernel, the columns that are left by the other one,
    // launched behind it (512 x 28672 x 8192, 3 rounds and 2 tiles of 256 x 256).
    const uint64_t rest = tiles_m * tiles_n % (sms / 2), strip = rest ? (rest + tiles_m - 1) / tiles_m : 0;
    if (swap_fits && strip && strip < tiles_n) {
        const uint32_t n0 = (uint32_t)(tiles_n - strip) * 256;
        const uint64_t both = pair_price(tiles_m * (tiles_n - strip), ktiles, sms) + swap_price(M, blocks_m * cdiv(N - n0, 128), ktiles, sms) + 160;
        if (both < one) return n0;
    }
    return swap < pairs ? 0 : N;
}
template <int FMT, class T>
static int gemm(const GemmArgs &a, cudaStream_t st, uint32_t early) {
    const uint32_t n0 = a.M <= 128 ? 0 : pair_columns(a.M, a.N, a.K, (uint64_t)sm_count_current_device());
    if (n0 == 0) return launch_swap<FMT, T>(a, st, early);
    if (n0 == a.N) return launch_pair<FMT, T>(a, st);
    GemmArgs main = a, left = a;
    main.N = n0;
    left.N = a.N - n0;
    left.w += (size_t)n0 * (a.K / 2);
    left.w_scales += (size_t)(n0 / 128) * scale_tiles(FMT, a.K) * kTileBytes;
    if (a.w_rows) left.w_rows += n0;
    if (a.bias) left.bias = reinterpret_cast<const uint16_t *>(a.bias) + n0;
    left.out = reinterpret_cast<uint16_t *>(a.out) + n0;
    const int rc = launch_pair<FMT, T>(main, st);
    return rc ? rc : launch_swap<FMT, T>(left, st, 2);
}

static int check_gemm(int format, int dtype, uint32_t M, uint32_t N, uint32_t K, uint64_t ldo) {
    if (format != kMX && format != kNV) return DUQ4_ERR_MODE;
    if (dtype != DUQ4_DTYPE_F16 && dtype != DUQ4_DTYPE_BF16) return DUQ4_ERR_MODE;
    if (K == 0 || K % 32 != 0 || ldo < N || (M | N | K) > 0x7FFFFFFFu) return DUQ4_ERR_SHAPE;
    return DUQ4_OK;
}
static bool aligned(const void *p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

static int run(int format, int dtype, const GemmArgs &a, cudaStream_t st, uint32_t early) {
    if (format == kMX) return dtype == DUQ4_DTYPE_F16 ? gemm<kMX, __half>(a, st, early) : gemm<kMX, __nv_bfloat16>(a, st, early);
    return dtype == DUQ4_DTYPE_F16 ? gemm<kNV, __half>(a, st, early) : gemm<kNV, __nv_bfloat16>(a, st, early);
}

static size_t up256(size_t v) { return (v + 255) / 256 * 256; }

}  // namespace fp4

int fp4_status_read(int32_t *out) {
    int v = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&v, g_fp4_status, sizeof(int));
    if (e != cudaSuccess) return (int)e;
    *out = v;
    if (v != 0) {
        int zero = 0;
        cudaMemcpyToSymbol(g_fp4_status, &zero, sizeof(int));
    }
    return DUQ4_OK;
}

}  // namespace duq4

using namespace duq4;
using namespace duq4::fp4;

extern "C" {

int duq4_linear_fp4(int format, const uint8_t *A, const uint8_t *A_block_scales, const float *A_row_scales, const uint8_t *W,
                    const uint8_t *W_block_scales, const float *W_row_scales, uint32_t M, uint32_t N, uint32_t K, const void *bias, int dtype,
                    void *out, uint64_t ldo, void *stream) {
    DUQ4_TRACE();
    if (ldo == 0) ldo = N;
    int rc = check_gemm(format, dtype, M, N, K, ldo);
    if (rc) return rc;
    if (M == 0 || N == 0) return DUQ4_OK;
    if (!A || !A_block_scales || !W || !W_block_scales || !out) return DUQ4_ERR_NULL;
    if (!aligned(A, 16) || !aligned(A_block_scales, 16) || !aligned(W, 16) || !aligned(W_block_scales, 16) || !aligned(A_row_scales, 4) ||
        !aligned(W_row_scales, 4) || !aligned(bias, 2) || !aligned(out, 2))
        return DUQ4_ERR_ALIGN;
    const GemmArgs a{M, N, K, A, A_block_scales, W, W_block_scales, A_row_scales, W_row_scales, bias, out, ldo};
    return run(format, dtype, a, (cudaStream_t)stream, g_static_weights.load(std::memory_order_relaxed) ? 1 : 3);
}

int duq4_fp4_wait_selftest(int32_t *result, void *stream) {
    DUQ4_TRACE();
    if (!result) return DUQ4_ERR_NULL;
    if (!aligned(result, 4)) return DUQ4_ERR_ALIGN;
    fp4_wait_selftest_kernel<<<1, 32, 0, (cudaStream_t)stream>>>(result);
    return launch_status();
}

uint32_t duq4_linear_fp4_pair_columns(uint32_t M, uint32_t N, uint32_t K, uint32_t sms) {
    return sms < 2 || M == 0 || N == 0 || K == 0 || (M | N | K) > 0x7FFFFFFFu ? 0 : pair_columns(M, N, K, sms);
}

size_t duq4_linear_fp4_workspace_bytes(int format, uint32_t M, uint32_t K) {
    return up256((size_t)M * (K / 2)) + up256(duq4_fp4_scale_bytes(format, M, K)) + up256((size_t)M * 4);
}

int duq4_linear_fp4_from_16bit(int format, int dtype, const void *x, const uint8_t *W, const uint8_t *W_block_scales,
                               const float *W_row_scales, uint32_t M, uint32_t N, uint32_t K, const void *bias, void *out, uint64_t ldo,
                               void *workspace, size_t workspace_bytes, void *stream) {
    DUQ4_TRACE();
    if (ldo == 0) ldo = N;
    int rc = check_gemm(format, dtype, M, N, K, ldo);
    if (rc) return rc;
    if (M == 0 || N == 0) return DUQ4_OK;
    if (!x || !W || !W_block_scales || !out) return DUQ4_ERR_NULL;
    if (!workspace || !aligned(workspace, 256) || workspace_bytes < duq4_linear_fp4_workspace_bytes(format, M, K)) return DUQ4_ERR_WORKSPACE;
    if (!aligned(W, 16) || !aligned(W_block_scales, 16) || !aligned(W_row_scales, 4) || !aligned(bias, 2) || !aligned(out, 2)) return DUQ4_ERR_ALIGN;
    uint8_t *codes = (uint8_t *)workspace, *scales = codes + up256((size_t)M * (K / 2));
    float *rows = format == kNV ? (float *)(scales + up256(duq4_fp4_scale_bytes(format, M, K))) : nullptr;
    rc = fp4_quantize_rows(format, dtype, x, M, K, K, codes, scales, rows, (cudaStream_t)stream);
    if (rc) return rc;
    const GemmArgs a{M, N, K, codes, scales, W, W_block_scales, rows, W_row_scales, bias, out, ldo};
    // The product may start while the quantizer runs: the quantizer lets it only when everything that was queued before (the
    // weights' upload among it) is done; what the quantizer writes itself is waited for in the kernel.
    return run(format, dtype, a, (cudaStream_t)stream, 1);
}

}  // extern "C"
