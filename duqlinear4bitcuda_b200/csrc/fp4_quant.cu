// Quantizers of the microscaled 4-bit formats and the operators that end in one: activations as they are, the SiLU-gated
// product of a gate/up projection, and the residual sum between two blocks with its norms. One row kernel does all three:
// a row is formed in registers, 16 neighbours per thread, and coded from there, so that no intermediate goes to memory.
// No counterpart in the reference, whose quantizers are integer ones (qlinear4bit/nn/quantizer.py).
#include <type_traits>

#include "fp4_common.cuh"
#include "quant_device.cuh"
#include "trace_range.h"

namespace duq4 {
namespace fp4 {

enum { SRC_PLAIN, SRC_SILU, SRC_NORM };
enum { OUT_ROW = DUQ4_MODE_NONE, OUT_SYM = DUQ4_MODE_SYM, OUT_ASYM = DUQ4_MODE_ASYM, OUT_MX = kMX, OUT_NV = kNV };

struct RowArgs {
    uint32_t rows, cols;
    uint64_t ldx;                 // elements between rows of x
    const uint16_t *x;            // SRC_SILU: gate and up projections side by side
    uint32_t up_offset;
    // SRC_NORM
    const uint16_t *residual, *post_weight, *gate, *weight;
    uint16_t *residual_out;
    uint32_t gate_per_row;
    float residual_scale;
    double eps, inv_cols;         // 1 / cols
    float clip;
    // results
    uint8_t *codes;               // OUT_ROW: the 16-bit row itself
    uint8_t *block_scales;        // OUT_SYM / OUT_ASYM: fp16 scales [rows]
    void *row_scales;             // OUT_NV: float [rows]; OUT_ASYM: fp16 zero-points [rows]
    uint32_t lanes;               // threads of a row (narrow rows)
    uint32_t wide;                // every 16-bit tensor and row starts on a 32-byte boundary
};

struct Chunk {                    // 16 neighbours of a row
    uint32_t w[8];
};
// Plain (not read-only-path) accesses: the norm's tensors may be written in place.
__device__ __forceinline__ Chunk load_chunk(const uint16_t *p, bool wide) {
    Chunk c;
    if (wide) {
        asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(c.w[0]), "=r"(c.w[1]), "=r"(c.w[2]), "=r"(c.w[3]), "=r"(c.w[4]), "=r"(c.w[5]), "=r"(c.w[6]), "=r"(c.w[7])
                     : "l"(p));
    } else {
        const uint4 a = reinterpret_cast<const uint4 *>(p)[0], b = reinterpret_cast<const uint4 *>(p)[1];
        c.w[0] = a.x; c.w[1] = a.y; c.w[2] = a.z; c.w[3] = a.w;
        c.w[4] = b.x; c.w[5] = b.y; c.w[6] = b.z; c.w[7] = b.w;
    }
    return c;
}
__device__ __forceinline__ void store_chunk(uint16_t *p, const Chunk &c, bool wide) {
    if (wide) {
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(c.w[0]), "r"(c.w[1]), "r"(c.w[2]), "r"(c.w[3]),
                     "r"(c.w[4]), "r"(c.w[5]), "r"(c.w[6]), "r"(c.w[7]) : "memory");
    } else {
        reinterpret_cast<uint4 *>(p)[0] = make_uint4(c.w[0], c.w[1], c.w[2], c.w[3]);
        reinterpret_cast<uint4 *>(p)[1] = make_uint4(c.w[4], c.w[5], c.w[6], c.w[7]);
    }
}

// Two floats per instruction, each rounded as by itself.
struct Pair2 {
    uint64_t v;
};
__device__ __forceinline__ Pair2 pair2(float2 f) {
    Pair2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(f.x), "f"(f.y));
    return r;
}
__device__ __forceinline__ Pair2 both(float f) { return pair2(make_float2(f, f)); }
__device__ __forceinline__ float2 unpair(Pair2 p) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p.v));
    return f;
}
__device__ __forceinline__ Pair2 add2(Pair2 a, Pair2 b) {
    Pair2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Pair2 mul2(Pair2 a, Pair2 b) {
    Pair2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Pair2 fma2(Pair2 a, Pair2 b, Pair2 c) {
    Pair2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
// -x / d for two quotients: by minus the approximate reciprocal of d, then one step of iterative refinement,
// q + (x + q d) ninv with q = -x / d nearly. The residual is exact (fma), so what is left of the reciprocal's error is about its
// square: where q and d are normal numbers the result is off by half a unit and 2^-21 of one at most, the nearest float but for
// quotients that near to the middle of two. The coding below has none (see there); of the SiLU quotient the tests compare
// every 16-bit gate. (The negated quotient, because then a zero keeps its sign without an instruction for it.)
__device__ __forceinline__ Pair2 minus_quotient2(Pair2 x, Pair2 d, Pair2 ninv) {
    const Pair2 q = mul2(x, ninv);
    return fma2(fma2(q, d, x), ninv, q);
}

// h = silu(g) * u with the roundings of F.silu(gate) * up on 16-bit tensors: silu in 32 bits, rounded, then the product. (The
// rounded silu equals torch's for each of the 65536 gates of either type, beside whatever gate it is paired with.)
template <class T>
__device__ __forceinline__ uint32_t silu_mul_two(uint32_t g, uint32_t u) {
    const float2 x = Two<T>::up(g), y = Two<T>::up(u);
    float2 s;
    const float2 d = make_float2(1.0f + expf(-x.x), 1.0f + expf(-x.y));
    if (fmaxf(fabsf(x.x), fabsf(x.y)) < 80.f)   // d below 6e34 (a NaN beside a number passes and stays one)
        s = unpair(minus_quotient2(pair2(x), pair2(d), pair2(make_float2(rcp_approx_ftz(-d.x), rcp_approx_ftz(-d.y)))));
    else
        s = make_float2(-__fdiv_rn(x.x, d.x), -__fdiv_rn(x.y, d.y));
    s = unpair(mul2(pair2(Two<T>::up(Two<T>::down(s.x, s.y))), pair2(y)));
    return Two<T>::down(s.x, s.y) ^ 0x80008000u;
}

// Sums and maxima over the threads of a row (the block, or `nt` lanes of a warp); every thread gets the result. `sm` must not
// be in use by an earlier reduction's readers.
template <bool LANES>
__device__ __forceinline__ double row_sum(double v, uint32_t nt, double *sm) {
    if (LANES) {
        for (uint32_t o = nt >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    }
    const uint32_t lane = threadIdx.x & 31, warps = nt >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (warps == 1) return v;
    if (lane == 0) sm[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < warps ? sm[lane] : 0.0;
    for (uint32_t o = warps > 16 ? 16 : warps > 8 ? 8 : warps > 4 ? 4 : 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return __shfl_sync(0xffffffffu, v, 0);
}
template <bool LANES>
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t nt, uint32_t *sm) {
    if (LANES) {
        for (uint32_t o = nt >> 1; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
        return v;
    }
    const uint32_t lane = threadIdx.x & 31, warps = nt >> 5;
    v = __reduce_max_sync(0xffffffffu, v);
    if (warps == 1) return v;
    if (lane == 0) sm[threadIdx.x >> 5] = v;
    __syncthreads();
    return __reduce_max_sync(0xffffffffu, lane < warps ? sm[lane] : 0u);
}

template <class T>
__device__ __forceinline__ uint32_t chunk_top(const Chunk &c) {   // largest magnitude's bits (above kInf: a NaN)
    uint32_t m = Two<T>::abs_max(c.w[0], c.w[1]);
#pragma unroll
    for (int k = 2; k < 8; ++k) m = Two<T>::abs_max(m, c.w[k]);
    m &= 0x7FFF7FFFu;
    return max(m & 0xFFFFu, m >> 16);
}

// 1 / sqrt(mean of squares + eps) of the row that the block's threads hold. Codes jump at borders and must not depend on
// the order of a sum, so the sum is carried with its rounding errors. Squares of 16-bit values are exact in 32 bits; a
// thread's sum S starts at a power of two beyond its largest square, so that in S' = S + x^2 the part that S takes,
// S' - S, is exact and so is the rest, x^2 - (S' - S), which is summed beside it (Dekker's fast two-sum): four
// operations a value, and an error of the square of a rounding (emulated, normal rows: 6e-16 of the sum at most; the bound for
// 32 values a thread, all of a sign and size for it, is 2^-34). The threads' sums meet in 64 bits. Rows whose squares
// leave the range of 32 bits (bfloat16 beyond 1e18 or below 1e-15, infinities, NaNs) are summed in 64 bits instead.
// `again`: where the thread, tid of the row's nt, finds its row once more for that.
template <class T, int CH, bool LANES>
__device__ __forceinline__ float row_rstd(const Chunk (&d)[CH], const RowArgs &a, const uint16_t *again, uint32_t tid, uint32_t nt, double *sm) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < CH; ++i) top = max(top, chunk_top<T>(d[i]));
    const float m = Two<T>::up1(top), m2 = m * m;
    const float start = __uint_as_float((__float_as_uint(m2) & 0x7F800000u) + 0x01000000u);   // in (2 m^2, 4 m^2]
    const bool odd = top != 0 && !(m2 > 1e-30f && m2 < 1e36f);
    const Pair2 minus_one = both(-1.f);
    Pair2 s = both(start), c = both(0.f);
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) {   // chunks beyond the row's end hold zeros
            const Pair2 x = pair2(Two<T>::up(d[i].w[k]));
            const Pair2 t = fma2(x, x, s);
            c = add2(c, fma2(x, x, fma2(t, minus_one, s)));
            s = t;
        }
    const float2 sf = unpair(s), cf = unpair(c);
    double sum = ((double)(sf.x - start) + (double)(sf.y - start)) + ((double)cf.x + (double)cf.y);   // sf - start is exact
    if (odd) {
        sum = 0;
#pragma unroll 1
        for (uint32_t c = tid; c < a.cols >> 4; c += nt)
#pragma unroll 1
            for (int k = 0; k < 8; ++k) {
                const float2 x = Two<T>::up(reinterpret_cast<const volatile uint32_t *>(again + c * 16)[k]);
                sum += (double)x.x * x.x + (double)x.y * x.y;
            }
    }
    const double v = row_sum<LANES>(sum, nt, sm) * a.inv_cols + a.eps;
    if (!(v > 1e-30 && v < 1e30)) return (float)(1.0 / sqrt(v));
    // One step of third order in 64 bits from the 32-bit root r, which is off by e < 2^-21.8 relative: with h = 1 - v r^2, about
    // 2e, the exact root is r (1 + h/2 + 3/8 h^2 + ...), and the next term is below 2^-64. What is left are the roundings of these
    // operations, below 2^-51 together. (A step of second order leaves 1.5 e^2, up to 1e-13: seen in the result's last bit.)
    const double r = (double)rsqrtf((float)v), h = 1.0 - v * r * r;
    return (float)(r + r * h * (0.5 + 0.375 * h));
}

// CH chunks per thread. A row is a CTA's, or -- LANES, narrow rows -- that of `lanes` (8, 16 or 32) lanes of a warp, which
// need no barrier to meet.
template <int SRC, class T, int OUT, int CH, bool LANES, int REGS>
__global__ void __maxnreg__(REGS) fp4_row_kernel(const RowArgs a) {
    __shared__ double sm_d[2][32];
    __shared__ uint32_t sm_u[32];
    __shared__ float sm_f[32][4];
    const uint32_t chunks_all = a.cols >> 4, NT = LANES ? a.lanes : blockDim.x, tid = LANES ? threadIdx.x & (NT - 1) : threadIdx.x;
    const int lane = threadIdx.x & 31;
    const bool wide = a.wide != 0;
    // This launch may begin while the one in front ends; it waits here, before its first access to memory. Only then may the
    // next one begin (a product, which fetches its weights while these rows are coded): all that was queued earlier is done.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // LANES: a warp's rows are neighbours; it goes on together until none of them exists
    const uint32_t per_warp = LANES ? 32 / NT : 1, mine = LANES ? lane / NT : 0;
    const uint32_t first = LANES ? (blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)) * per_warp : blockIdx.x;
    const uint32_t step = LANES ? gridDim.x * (blockDim.x >> 5) * per_warp : gridDim.x;
    for (uint64_t at = first; at < a.rows; at += step) {
        const bool there = at + mine < a.rows;
        const uint32_t row = there ? (uint32_t)(at + mine) : a.rows - 1, chunks = there ? chunks_all : 0;
        Chunk d[CH];
        const uint16_t *xr = a.x + (size_t)row * a.ldx;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const uint32_t c = tid + i * NT;
            if (c < chunks) {
                d[i] = load_chunk(xr + c * 16, wide);
                if (SRC == SRC_SILU) {
                    const Chunk u = load_chunk(xr + a.up_offset + c * 16, wide);
#pragma unroll
                    for (int k = 0; k < 8; ++k) d[i].w[k] = silu_mul_two<T>(d[i].w[k], u.w[k]);
                }
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) d[i].w[k] = 0;
            }
        }
        if (SRC == SRC_NORM) {
            const size_t base = (size_t)row * a.cols;
            if (a.residual) {
                float rstd = 1.f;
                if (a.post_weight) rstd = row_rstd<T, CH, LANES>(d, a, xr, tid, NT, sm_d[0]);
#pragma unroll
                for (int i = 0; i < CH; ++i) {
                    const uint32_t c = tid + i * NT;
                    if (c >= chunks) continue;
                    const Chunk r = load_chunk(a.residual + base + c * 16, wide);
                    Pair2 y[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) y[k] = pair2(Two<T>::up(d[i].w[k]));
                    if (a.post_weight) {
                        const Chunk w = load_chunk(a.post_weight + c * 16, wide);
#pragma unroll
                        for (int k = 0; k < 8; ++k) y[k] = mul2(mul2(y[k], both(rstd)), pair2(Two<T>::up(w.w[k])));
                    }
                    if (a.gate) {
                        const Chunk w = load_chunk(a.gate + (a.gate_per_row ? base : 0) + c * 16, wide);
#pragma unroll
                        for (int k = 0; k < 8; ++k) y[k] = mul2(y[k], pair2(Two<T>::up(w.w[k])));
                    }
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        // one by one: a two-float product and a two-float sum behind it are contracted into an fma
                        const float2 yk = unpair(y[k]), rk = Two<T>::up(r.w[k]);
                        d[i].w[k] = Two<T>::down(__fadd_rn(rk.x, __fmul_rn(yk.x, a.residual_scale)), __fadd_rn(rk.y, __fmul_rn(yk.y, a.residual_scale)));
                    }
                    store_chunk(a.residual_out + base + c * 16, d[i], wide);
                }
            }
            const float rstd = row_rstd<T, CH, LANES>(d, a, a.residual ? a.residual_out + base : xr, tid, NT, sm_d[1]);
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                const uint32_t c = tid + i * NT;
                if (c >= chunks) continue;
                const Chunk w = load_chunk(a.weight + c * 16, wide);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float2 o = unpair(mul2(mul2(pair2(Two<T>::up(d[i].w[k])), both(rstd)), pair2(Two<T>::up(w.w[k]))));
                    d[i].w[k] = Two<T>::down(o.x, o.y);
                }
            }
        }
        if (OUT == OUT_ROW) {
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                const uint32_t c = tid + i * NT;
                if (c < chunks) store_chunk(reinterpret_cast<uint16_t *>(a.codes) + (size_t)row * a.cols + c * 16, d[i], wide);
            }
        } else if constexpr (OUT == OUT_SYM || OUT == OUT_ASYM) {
            static_assert(!LANES, "the integer formats' statistics meet in the block");
            // the framework's integer formats: statistics, scale and codes of quant_fused_vec_kernel on the row h
            constexpr int MODE = OUT == OUT_SYM ? QSYM : QASYM;
            Stats st;
            stats_init<MODE>(st);
            uint32_t am = 0;
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                if (tid + i * NT >= chunks) continue;
                am = max(am, chunk_top<T>(d[i]));
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float2 x = Two<T>::up(d[i].w[k]);
                    stats_add<MODE>(st, x.x, 16);
                    stats_add<MODE>(st, x.y, 16);
                }
            }
            const bool special = __syncthreads_or(am >= Two<T>::kInf);
            stats_reduce<MODE>(st, sm_f);
            const RowQ r = rowq_from_stats<MODE>(st, a.clip);
            __half *s1 = reinterpret_cast<__half *>(a.block_scales), *z1 = reinterpret_cast<__half *>(a.row_scales);
            if (threadIdx.x == 0) store_rowq<MODE>(r, row, s1, z1, nullptr, nullptr);
            const FastQ fq = make_fastq<MODE>(r, special);
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                const uint32_t c = tid + i * NT;
                if (c >= chunks) continue;
                const uint4 lo = make_uint4(d[i].w[0], d[i].w[1], d[i].w[2], d[i].w[3]);
                const uint4 hi = make_uint4(d[i].w[4], d[i].w[5], d[i].w[6], d[i].w[7]);
                uint2 q;
                q.x = fq.ok ? code8_fast<MODE>(lo, fq) : code8<MODE>(lo, 16, r);
                q.y = fq.ok ? code8_fast<MODE>(hi, fq) : code8<MODE>(hi, 16, r);
                *reinterpret_cast<uint2 *>(a.codes + (size_t)row * (a.cols >> 1) + c * 8) = q;
            }
        } else {
            constexpr int FMT = OUT == OUT_NV ? kNV : kMX;
            uint8_t *codes = a.codes + (size_t)row * (a.cols >> 1);
            uint8_t *scales = a.block_scales + scale_offset(scale_tiles(FMT, a.cols), row, 0);
            float row_scale = 1.f, six = 6.f, inv6 = 0.f;
            if (FMT == kNV) {
                uint32_t top = 0;   // over the blocks without infinities and NaNs
#pragma unroll
                for (int i = 0; i < CH; ++i) {
                    const uint32_t t = chunk_top<T>(d[i]);
                    if (t < Two<T>::kInf) top = max(top, t);
                }
                top = row_max<LANES>(top, NT, sm_u);
                // 8 bits, so that 6 * row_scale and block scale * row_scale are exact
                row_scale = __bfloat162float(__float2bfloat16_rn(__fdiv_rn(Two<T>::up1(top), 2688.f)));
                row_scale = fmaxf(row_scale, 7.703719777548943e-34f);   // 2^-110
                if (tid == 0 && there) reinterpret_cast<float *>(a.row_scales)[row] = row_scale;
                six = 6.f * row_scale;
                inv6 = __fdiv_rn(1.f, six);
            }
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                const uint32_t c = tid + i * NT;
                uint32_t top = chunk_top<T>(d[i]);
                if (FMT == kMX) top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                const bool special = top >= Two<T>::kInf;
                uint32_t scale;
                float q[2][8];
                if (FMT == kMX) {
                    // 2^(floor(log2 top) - 2): the exponent field of the float, less 2
                    const int e = max((int)(__float_as_uint(Two<T>::up1(top)) >> 23) - 2, 0);
                    const float inv = special ? 0.f : __uint_as_float((uint32_t)(254 - e) << 23);
                    const Pair2 inv2 = both(inv);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const float2 y = unpair(mul2(pair2(Two<T>::up(d[i].w[k])), inv2));
                        q[k >> 2][2 * (k & 3)] = y.x;
                        q[k >> 2][2 * (k & 3) + 1] = y.y;
                    }
                    scale = special ? 0xFFu : (uint32_t)e;
                } else {
                    // top / (6 row_scale): the middle of two e4m3 numbers exactly or at least 2^-15 away from it, so the
                    // refined quotient rounds as the exact one
                    const float t = Two<T>::up1(top), t0 = __fmul_rn(t, inv6);
                    scale = special ? 0x7Fu : e4m3_of(__fmaf_rn(__fmaf_rn(-t0, six, t), inv6, t0));
                    const float dd = special ? 0.f : __fmul_rn(e4m3_to_float(scale), row_scale);
                    const float inv = dd > 0.f ? rcp_approx_ftz(dd) : 0.f;
                    // x / dd, a 16-bit value by a 12-bit one: as far from the middles of two codes
                    const Pair2 dd2 = both(dd), ninv2 = both(-inv);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const float2 y = unpair(minus_quotient2(pair2(Two<T>::up(d[i].w[k])), dd2, ninv2));
                        q[k >> 2][2 * (k & 3)] = y.x;
                        q[k >> 2][2 * (k & 3) + 1] = y.y;
                    }
                }
                if (c >= chunks) scale = 0;   // padding blocks of the last scale tile
                if (c < chunks) {
                    uint2 w;
                    const uint32_t keep = special ? 0u : 0xFFFFFFFFu;   // (a bad block's quotients are NaNs)
                    w.x = (e2m1x8(q[0]) ^ (FMT == kNV ? 0x88888888u : 0u)) & keep;
                    w.y = (e2m1x8(q[1]) ^ (FMT == kNV ? 0x88888888u : 0u)) & keep;
                    *reinterpret_cast<uint2 *>(codes + c * 8) = w;
                }
                // four block scales are one word of a tile, stored by the first lane of the 8 (4) that hold them
                constexpr int kStep = FMT == kMX ? 2 : 1;
                scale |= __shfl_down_sync(0xffffffffu, scale, kStep) << 8;
                scale |= __shfl_down_sync(0xffffffffu, scale, 2 * kStep) << 16;
                if ((lane & (4 * kStep - 1)) == 0 && c < chunks)
                    *reinterpret_cast<uint32_t *>(scales + c / (4 * kStep) * 512) = scale;
            }
        }
        if (!LANES) __syncthreads();   // the reductions' buffers are free for the next row
    }
}

// Codes back to values: code * (block scale * row scale), rounded once. One thread per 16 neighbours. (No read-only-path
// loads, which need not stay behind the wait.)
template <int FMT, class T>
__global__ void __launch_bounds__(256) fp4_dequant_kernel(const uint8_t *codes, const uint8_t *scales, const float *row_scales, uint32_t rows,
                                                          uint32_t cols, T *out, bool wide) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t chunks = cols >> 4, tiles = scale_tiles(FMT, cols);
    const uint64_t total = (uint64_t)rows * chunks;
    for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (uint64_t)gridDim.x * blockDim.x) {
        const uint32_t row = (uint32_t)(i / chunks), c = (uint32_t)(i % chunks), blk = FMT == kMX ? c >> 1 : c;
        float s = block_scale_to_float<FMT>(scales[scale_offset(tiles, row, blk >> 2) + (blk & 3)]);
        if (FMT == kNV) s = __fmul_rn(s, row_scales[row]);
        const uint2 w = *reinterpret_cast<const uint2 *>(codes + i * 8);
        float v[16];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float2 f = __half22float2(e2m1x2_to_half2((k < 4 ? w.x : w.y) >> (8 * (k & 3)) & 0xFFu));
            v[2 * k] = __fmul_rn(f.x, s);
            v[2 * k + 1] = __fmul_rn(f.y, s);
        }
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                reinterpret_cast<float4 *>(out + i * 16)[k] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
        } else {
            Chunk o;
#pragma unroll
            for (int k = 0; k < 8; ++k) o.w[k] = Two<T>::down(v[2 * k], v[2 * k + 1]);
            store_chunk(reinterpret_cast<uint16_t *>(out + i * 16), o, wide);
        }
    }
}

static bool aligned(const void *p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// 16 neighbours per thread and chunk; rows of up to 65536 stay in registers.
constexpr uint32_t kMaxCols = 65536;

// A launch that may begin while the one in front on the stream ends (its kernel waits for that).
template <class... P, class... A>
static int launch_behind(uint32_t grid, uint32_t threads, cudaStream_t st, void (*kernel)(P...), A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, P(args)...);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return (int)e;
    }
    return launch_status();
}

template <int SRC, class T, int OUT>
static int launch_rows(RowArgs a, cudaStream_t st) {
    const uint32_t chunks = a.cols >> 4;
    const uint32_t grid = a.rows < 148u * 64u ? a.rows : 148u * 64u;
    a.inv_cols = 1.0 / a.cols;
    uintptr_t bits = reinterpret_cast<uintptr_t>(a.x) | (uintptr_t)(a.ldx * 2) | (uintptr_t)a.up_offset * 2 | reinterpret_cast<uintptr_t>(a.residual) |
                     reinterpret_cast<uintptr_t>(a.residual_out) | reinterpret_cast<uintptr_t>(a.post_weight) | reinterpret_cast<uintptr_t>(a.gate) |
                     reinterpret_cast<uintptr_t>(a.weight);
    if (OUT == OUT_ROW) bits |= reinterpret_cast<uintptr_t>(a.codes);
    a.wide = (bits & 31) == 0;
    auto threads = [&](uint32_t ch) { return cdiv(cdiv(chunks, ch), 32) * 32; };
    // Few rows: 16 columns per thread, so that a row is done soonest (1 x 4096, norm: 2.4 us against 2.6 with 32). Many rows:
    // 32, so that the reductions' fixed cost is spread (4096 x 8192, norm: 29 us against 38 with 16 and 33 with 64). Wide
    // rows without a norm, whose registers allow it: 64, so that two rows fit an SM and one loads while the other computes
    // (us with 32 / 64, nvfp4: 4096 x 8192 18.7 / 16.4, 2048 x 11008 17.1 / 13.5, 1024 x 28672 23.3 / 17.7, silu 2048 x 11008
    // 35.8 / 31.5, 4096 x 8192 40.1 / 41.8; mxfp4: 2048 x 11008 10.8 / 10.7, silu 26.3 / 28.4, 2048 x 16384 15.9 / 13.9, silu
    // 38.3 / 36.9; norm joint, 2048 x 16384: 55.3 / 60.6).
    constexpr uint32_t kWide = SRC == SRC_NORM ? 2048 : OUT != OUT_NV ? 768 : SRC == SRC_PLAIN ? 256 : 512;
    // Narrow rows, and enough of them for every SM: lanes of a warp (us with CTAs / lanes, mxfp4: 65536 x 128 16.0 / 5.9, norm
    // joint 69.9 / 16.4; 32768 x 512 12.1 / 10.7, 38.6 / 32.0; wider rows on a warp, two or four chunks a lane, 16384 x 1024:
    // 11.2 / 8.4, 25.5 / 28.4; 8192 x 2048: 9.7 / 8.7, 26.9 / 35.1).
    if constexpr (OUT != OUT_SYM && OUT != OUT_ASYM) {
        if (chunks <= 32 && a.rows >= 296) {
            a.lanes = chunks <= 8 ? 8 : chunks <= 16 ? 16 : 32;
            const uint64_t blocks = ((uint64_t)a.rows * a.lanes + 255) / 256;
            return launch_behind(blocks < 148u * 64u ? (uint32_t)blocks : 148u * 64u, 256, st, fp4_row_kernel<SRC, T, OUT, 1, true, 64>, a);
        }
    }
    // Registers a thread may have: fewer where that puts more rows on an SM at little spilling (us with 64 / 56 / 48 / 40 at
    // 32 columns a thread: mxfp4 4096 x 11008 20.8 / 21.0 / 20.8 / 19.0, silu 60.4 / 50.1 / 50.0 / 46.3; nvfp4 silu 4096 x 8192
    // 41.1 / 40.9 / 38.9 / 39.0; norm joint 4096 x 11008, whose 352 threads fit twice with 64, three times with 48:
    // 88.1 / 79.6 / 78.0 / 105.8, but 2048 x 16384 56.4 / 60.8 / 60.4 / 82.4).
    if (a.rows < 296 && chunks <= 1024) {
        return launch_behind(grid, threads(1), st, fp4_row_kernel<SRC, T, OUT, 1, false, 64>, a);
    } else if (chunks <= kWide) {
        const uint32_t nt = threads(2);
        constexpr int kRegs = SRC == SRC_NORM ? 64 : OUT == OUT_MX ? 40 : SRC == SRC_SILU ? 48 : 64;
        if (SRC == SRC_NORM && 1024 / nt * nt < 768) return launch_behind(grid, nt, st, fp4_row_kernel<SRC, T, OUT, 2, false, SRC == SRC_NORM ? 48 : kRegs>, a);
        return launch_behind(grid, nt, st, fp4_row_kernel<SRC, T, OUT, 2, false, kRegs>, a);
    }
    return launch_behind(grid, threads(4), st, fp4_row_kernel<SRC, T, OUT, 4, false, 64>, a);
}

static int check_fp4(int format, int dtype, uint32_t cols) {
    if (format != kMX && format != kNV) return DUQ4_ERR_MODE;
    if (dtype != DUQ4_DTYPE_F16 && dtype != DUQ4_DTYPE_BF16) return DUQ4_ERR_MODE;
    if (cols == 0 || cols % 32 != 0 || cols > kMaxCols) return DUQ4_ERR_SHAPE;
    return DUQ4_OK;
}

template <int SRC>
static int quantize_rows(int format, int dtype, const RowArgs &a, cudaStream_t st) {
    if (format == kMX) return dtype == DUQ4_DTYPE_F16 ? launch_rows<SRC, __half, OUT_MX>(a, st) : launch_rows<SRC, __nv_bfloat16, OUT_MX>(a, st);
    return dtype == DUQ4_DTYPE_F16 ? launch_rows<SRC, __half, OUT_NV>(a, st) : launch_rows<SRC, __nv_bfloat16, OUT_NV>(a, st);
}

}  // namespace fp4

// duq4_fp4_quantize without its trace range: also the first half of duq4_linear_fp4_from_16bit.
int fp4_quantize_rows(int format, int dtype, const void *x, uint32_t rows, uint32_t cols, uint64_t ldx, uint8_t *codes,
                      uint8_t *block_scales, float *row_scales, cudaStream_t st) {
    using namespace fp4;
    int rc = check_fp4(format, dtype, cols);
    if (rc) return rc;
    if (rows == 0) return DUQ4_OK;
    if (!x || !codes || !block_scales || (format == kNV && !row_scales)) return DUQ4_ERR_NULL;
    if (ldx < cols || ldx % 8 != 0) return DUQ4_ERR_SHAPE;
    if (!aligned(x, 16) || !aligned(codes, 16) || !aligned(block_scales, 16) || !aligned(row_scales, 4)) return DUQ4_ERR_ALIGN;
    RowArgs a{};
    a.rows = rows; a.cols = cols; a.ldx = ldx;
    a.x = (const uint16_t *)x;
    a.codes = codes; a.block_scales = block_scales; a.row_scales = row_scales;
    return quantize_rows<SRC_PLAIN>(format, dtype, a, st);
}

}  // namespace duq4

using namespace duq4;
using namespace duq4::fp4;

extern "C" {

size_t duq4_fp4_scale_bytes(int format, uint32_t rows, uint32_t cols) {
    if (format != kMX && format != kNV) return 0;
    return ((size_t)rows + 127) / 128 * scale_tiles(format, cols) * 512;
}

int duq4_fp4_quantize(int format, int dtype, const void *x, uint32_t rows, uint32_t cols, uint64_t ldx, uint8_t *codes,
                      uint8_t *block_scales, float *row_scales, void *stream) {
    DUQ4_TRACE();
    return fp4_quantize_rows(format, dtype, x, rows, cols, ldx, codes, block_scales, row_scales, (cudaStream_t)stream);
}

int duq4_fp4_silu_mul_quantize(int format, int dtype, const void *gate_up, uint32_t rows, uint32_t inter, uint64_t ld, uint32_t up_offset,
                               uint8_t *codes, uint8_t *block_scales, float *row_scales, void *stream) {
    DUQ4_TRACE();
    int rc = check_fp4(format, dtype, inter);
    if (rc) return rc;
    if (rows == 0) return DUQ4_OK;
    if (!gate_up || !codes || !block_scales || (format == kNV && !row_scales)) return DUQ4_ERR_NULL;
    if (ld % 8 != 0 || up_offset % 8 != 0 || (uint64_t)up_offset + inter > ld) return DUQ4_ERR_SHAPE;
    if (!aligned(gate_up, 16) || !aligned(codes, 16) || !aligned(block_scales, 16) || !aligned(row_scales, 4)) return DUQ4_ERR_ALIGN;
    RowArgs a{};
    a.rows = rows; a.cols = inter; a.ldx = ld; a.up_offset = up_offset;
    a.x = (const uint16_t *)gate_up;
    a.codes = codes; a.block_scales = block_scales; a.row_scales = row_scales;
    return quantize_rows<SRC_SILU>(format, dtype, a, (cudaStream_t)stream);
}

int duq4_norm_residual_quantize(int format, const duq4_norm_residual *n, uint32_t rows, uint32_t cols, void *out, void *scales,
                                void *row_scales, void *stream) {
    DUQ4_TRACE();
    if (!n) return DUQ4_ERR_NULL;
    const bool integer = format == DUQ4_MODE_SYM || format == DUQ4_MODE_ASYM, floating = format == kMX || format == kNV;
    if (format != DUQ4_MODE_NONE && !integer && !floating) return DUQ4_ERR_MODE;
    int rc = check_fp4(kMX, n->dtype, cols);
    if (rc) return rc;
    if (integer && n->dtype != DUQ4_DTYPE_F16) return DUQ4_ERR_MODE;   // the integer formats' scales are fp16
    if (rows == 0) return DUQ4_OK;
    if (!n->x || !n->weight || !out || (format != DUQ4_MODE_NONE && !scales) || ((format == kNV || format == DUQ4_MODE_ASYM) && !row_scales))
        return DUQ4_ERR_NULL;
    if (n->residual ? !n->residual_out : (n->residual_out || n->post_weight || n->gate)) return DUQ4_ERR_NULL;
    if (!(n->eps >= 0)) return DUQ4_ERR_SHAPE;
    const void *must[] = {n->x, n->residual, n->residual_out, n->post_weight, n->gate, n->weight, out};
    for (const void *p : must)
        if (!aligned(p, 16)) return DUQ4_ERR_ALIGN;
    if (!aligned(scales, floating ? 16 : 2) || !aligned(row_scales, format == kNV ? 4 : 2)) return DUQ4_ERR_ALIGN;
    RowArgs a{};
    a.rows = rows; a.cols = cols; a.ldx = cols;
    a.x = (const uint16_t *)n->x;
    a.residual = (const uint16_t *)n->residual;
    a.residual_out = (uint16_t *)n->residual_out;
    a.post_weight = (const uint16_t *)n->post_weight;
    a.gate = (const uint16_t *)n->gate;
    a.gate_per_row = n->gate_per_row != 0;
    a.weight = (const uint16_t *)n->weight;
    a.residual_scale = n->residual_scale;
    a.eps = n->eps;
    a.clip = n->clip_ratio;
    a.codes = (uint8_t *)out;
    a.block_scales = (uint8_t *)scales;
    a.row_scales = row_scales;
    cudaStream_t st = (cudaStream_t)stream;
    if (format == DUQ4_MODE_SYM) return launch_rows<SRC_NORM, __half, OUT_SYM>(a, st);
    if (format == DUQ4_MODE_ASYM) return launch_rows<SRC_NORM, __half, OUT_ASYM>(a, st);
    if (format == DUQ4_MODE_NONE)
        return n->dtype == DUQ4_DTYPE_F16 ? launch_rows<SRC_NORM, __half, OUT_ROW>(a, st) : launch_rows<SRC_NORM, __nv_bfloat16, OUT_ROW>(a, st);
    return quantize_rows<SRC_NORM>(format, n->dtype, a, st);
}

int duq4_fp4_dequantize(int format, int dtype, const uint8_t *codes, const uint8_t *block_scales, const float *row_scales, uint32_t rows,
                        uint32_t cols, void *out, void *stream) {
    DUQ4_TRACE();
    if (format != kMX && format != kNV) return DUQ4_ERR_MODE;
    if (dtype != DUQ4_DTYPE_F16 && dtype != DUQ4_DTYPE_BF16 && dtype != DUQ4_DTYPE_F32) return DUQ4_ERR_MODE;
    if (cols == 0 || cols % 32 != 0) return DUQ4_ERR_SHAPE;
    if (rows == 0) return DUQ4_OK;
    if (!codes || !block_scales || !out || (format == kNV && !row_scales)) return DUQ4_ERR_NULL;
    if (!aligned(codes, 8) || !aligned(out, 16) || !aligned(row_scales, 4)) return DUQ4_ERR_ALIGN;
    cudaStream_t st = (cudaStream_t)stream;
    const uint64_t total = (uint64_t)rows * (cols >> 4);
    const uint32_t grid = (uint32_t)((total + 255) / 256 < 148u * 32u ? (total + 255) / 256 : 148u * 32u);
    int rc = DUQ4_OK;
    auto go = [&](auto fmt, auto *o) {
        auto *kernel = fp4_dequant_kernel<decltype(fmt)::value, std::remove_pointer_t<decltype(o)>>;
        rc = launch_behind(grid, 256, st, kernel, codes, block_scales, row_scales, rows, cols, o, aligned(out, 32));
    };
    auto by_type = [&](auto fmt) {
        if (dtype == DUQ4_DTYPE_F16) go(fmt, (__half *)out);
        else if (dtype == DUQ4_DTYPE_BF16) go(fmt, (__nv_bfloat16 *)out);
        else go(fmt, (float *)out);
    };
    if (format == kMX) by_type(std::integral_constant<int, kMX>{});
    else by_type(std::integral_constant<int, kNV>{});
    return rc;
}

}  // extern "C"
