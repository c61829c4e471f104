// A linear's weight gradient from an 8-bit checkpoint of its input, on the
// sm_100a tensor cores (tcgen05 kind::f16, fp32 accumulation in TMEM):
//
//   dw[n, k] = col[k] * sum_m dy[m, n] * row[m] * q[m, k] * s[m, k / 128]
//
// q, s: the checkpoint (groups of 128 columns with power-of-two scales); row
// and col (nullable) are a norm's 1/rms per token and its weight, for a linear
// that stands behind one: then q * s is the norm's input and nothing else of
// the norm's output has to be kept.
//
// The kept values are never written out: each CTA loads the bytes, widens them
// in shared memory and multiplies.  q * s has 7 bits and a power of two, so it is
// exact in bf16, whatever s; `row` goes to the other operand.
//   * bf16 dy without `row` goes from TMA to the tensor cores as it is.
//   * otherwise dy (times row, in fp32) is split into bf16 parts: 16-bit dy into
//     two (16 bits: exact without row, with it off by at most 2^-17 of a term; one
//     part would be off by up to 2^-8, as much as a bf16 result's own rounding), fp32 dy
//     into three (24 bits), the high part into one accumulator and the two small
//     ones into another.  fp16 dy is not multiplied as it is, since fp16 does not
//     hold what a checkpoint may: kept values reach from 2^-100 to fp32's largest.
//
// Tile: one or two groups of 128 checkpoint columns (a token has one scale in
// each) as the MMA's rows, BN columns of dy as its columns, both "MN-major" (a
// token's values are contiguous; tokens are the reduction).  The tokens are cut
// into slices so that tiles x slices fill the GPU; a slice's tile goes to a
// workspace and w8_sum_kernel adds the slices in a fixed order.  Persistent, one
// CTA per SM, roles in separate warps over two rings of token blocks, one of
// blocks as they are loaded and one of widened ones: producer (TMA), the tokens'
// factors (cp.async), MMA issuer, converters, epilogue.  Every wait is bounded.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "tc_common.cuh"

namespace mmb {

constexpr int W8_BK = 128;  // checkpoint columns of a group
constexpr uint32_t W8_SWZ128 = 2;

// MMA of bf16 operands, both MN-major, fp32 accumulation: M = 128, N = n
__host__ __device__ constexpr uint32_t w8_idesc(int n) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | (1u << 16) |
           ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// alo, blo: the low words of the operands' descriptors; they share the high one
__device__ __forceinline__ void umma_f16(uint32_t d_tmem, uint32_t alo, uint32_t blo, uint32_t dhi,
                                         uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %3};\n\t"
        "mov.b64 db, {%2, %3};\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n\t}" ::"r"(d_tmem),
        "r"(alo), "r"(blo), "r"(dhi), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Operand layout of BT tokens: blocks of 64 columns, each BT rows (tokens) of
// 128 bytes with the 128-byte swizzle: 16-byte chunk c of token t lies at chunk
// c ^ (t % 8).  An MMA's step is 16 tokens on.
// In a descriptor's low word, 16 bytes count 1: the issuing thread adds offsets to
// words made once.
constexpr uint32_t W8_STEP = 16 * 128 / 16;
template <int BT>
__device__ __forceinline__ uint32_t w8_chunk(int block, int t, int c) {
    return (uint32_t)(block * (BT * 128) + t * 128 + ((c ^ (t & 7)) << 4));
}

// AG: checkpoint groups (128 columns) of a tile; BN: its dy columns; BT: tokens of
// a block; RL, RC: blocks in flight as they lie in memory / widened; RA:
// accumulators; CW, EW: converter (in CG groups, each at a block of its own) and
// epilogue warps.
//
// Two groups share each load of dy (65536 x (4096, 1024) bf16: 616 -> 477 us, in two
// parts 1241 -> 860).
//
// What bounds it is shared memory: a block of 64 tokens of a 256 x 256 tile moves
// 48 KB in by TMA, 16 KB out and 32 KB back through the converters and 96 KB into
// the tensor cores, 192 KB or 1536 cycles at 128 bytes a cycle, against 1024 cycles
// of MMAs.  B200: 65536 x (4096, 1024) bf16 466 us, slices added, 1.2e15 operations/s,
// 0.72 of the measured bf16 rate (400 us with the converters left out); 76800 x
// (1024, 256) bf16 61 us.  fp32, three parts: 76800 x (1024, 256) 165 us, 32768 x
// (512, 128) 29 us.  The plans of the large sizes give 128 units to 148 SMs.
template <int GROUPS>
struct W8Half {
    static constexpr bool F32 = false;
    static constexpr int PARTS = 1;  // dy as it is
    static constexpr int AG = GROUPS, BN = 256, BT = 64, BYTES = 2;
    static constexpr int RL = AG == 1 ? 4 : 3, RC = AG == 1 ? 3 : 2, RA = AG == 1 ? 2 : 1;
    static constexpr int CW = 8, CG = 1, EW = 8;
};
// The tensor cores' fp32 accumulation truncates: its error grows with the number
// of steps, so every so many tokens the sums leave TMEM and are added up with
// ordinary rounding.
//   * fp32 dy: 1024 tokens, added in registers, with the small parts in an
//     accumulator of their own: 2e-7 against 64 bits, nearer than an fp32 product.
//   * 16-bit dy, whose tiles are too large for registers: added where the result
//     goes, in fp32.  Against 64 bits, random values: an fp32 result of bf16 dy is off
//     by 1e-6 with 4096 tokens, 2.5e-6 with 8192 and 1.6e-5 with 32768, with dy in two
//     parts by 6e-6 with 4096 and 1.1e-5 with 8192; 65536 x (4096, 1024) takes 560 us,
//     505 and 470 (900 and 860).  A 16-bit result is off by its own 1.65e-3 or 2.05e-4
//     in any case and gathers 32768 tokens, in two parts (fp16 results) half of that.
constexpr int W8_SEG_FP32_DY = 1024, W8_SEG_FP32_DW = 4096, W8_SEG_16_DW = 32768;
struct W8F32 {
    static constexpr bool F32 = true;
    static constexpr int PARTS = 3;
    static constexpr int AG = 1, BN = 128, BT = 32, BYTES = 4;
    static constexpr int RL = 4, RC = 4, RA = 2, CW = 8, CG = 4, EW = 8;
};
// 16-bit dy (bf16 or fp16 in memory: BF) in two bf16 parts.  Blocks of 32 tokens
// leave room for both parts of 256 columns.  Twice the MMAs of W8Half, and dy goes
// through the converters: 65536 x (4096, 1024) bf16 852 us (one part 466), 76800 x
// (1024, 256) 84 us (61).  A block of 32 tokens and two groups moves what W8Half's of 64
// does, 192 KB against 1024 cycles of MMAs, and takes as long, 0.86 us.
template <bool BF, int GROUPS>
struct W8Two {
    static constexpr bool F32 = false;
    static constexpr int PARTS = 2;
    static constexpr int AG = GROUPS, BN = 256, BT = 32, BYTES = 2;
    static constexpr int RL = 3, RC = AG == 1 ? 4 : 3, RA = AG == 1 ? 2 : 1;
    static constexpr int CW = 8, CG = 2, EW = 8;
    // two values of dy in fp32
    static __device__ __forceinline__ float2 dy2(uint32_t w) {
        if constexpr (BF) return make_float2(bf16_lo(w), bf16_hi(w));
        else return __half22float2(*reinterpret_cast<const __half2*>(&w));
    }
};
template <class D>
struct W8Smem {
    static constexpr int DY = D::BT * D::BN * D::BYTES;  // dy as it lies in memory
    static constexpr int Q1 = D::BT * W8_BK;              // one group's bytes
    static constexpr int Q = D::AG * Q1;
    static constexpr int FACT = 1024;                    // scales and row factor of BT tokens
    static constexpr int LOAD = DY + Q + FACT;
    static constexpr int A1 = D::BT * W8_BK * 2;         // widened checkpoint, one group
    static constexpr int A = D::AG * A1;
    static constexpr int P1 = D::BT * D::BN * 2;          // one of dy's bf16 parts
    static constexpr int CONV = A + (D::PARTS > 1 ? D::PARTS * P1 : 0);
    static constexpr size_t BYTES = (size_t)D::RL * LOAD + (size_t)D::RC * CONV + 1024;
};
template <class D>
__host__ __device__ constexpr int w8_threads() { return 32 * (3 + D::CW + D::EW); }

__device__ __forceinline__ uint32_t w8_pack2(float a, float b) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&t);
}
// Two values as PARTS bf16 pairs whose sum they are.  From W8_EDGE on the nearest
// bf16 would be an infinity and the next part its opposite: the largest finite value
// is taken there, and an infinity or a NaN stands alone.
constexpr float W8_EDGE = 0x1.ffp127f, W8_BF16_MAX = 0x1.fep127f;
template <int PARTS>
__device__ __forceinline__ void w8_parts(float2 v, uint32_t (&o)[PARTS]) {
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
        o[i] = w8_pack2(v.x, v.y);
        v.x -= bf16_lo(o[i]);
        v.y -= bf16_hi(o[i]);
    }
}
template <int PARTS>
__device__ __forceinline__ void w8_parts_edge(float2 v, uint32_t (&o)[PARTS]) {
    const auto high = [](float x) {
        return fabsf(x) < INFINITY ? fminf(fmaxf(x, -W8_BF16_MAX), W8_BF16_MAX) : x;
    };
    const auto rest = [](float x, float h) { return fabsf(x) < INFINITY ? x - h : 0.f; };
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
        o[i] = w8_pack2(high(v.x), high(v.y));
        v.x = rest(v.x, bf16_lo(o[i]));
        v.y = rest(v.y, bf16_hi(o[i]));
    }
}
__device__ __forceinline__ float w8_top(float top, float2 v) {
    return fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y)));
}

// `bar` counts an arrival of this lane once its cp.async copies so far have landed
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}

struct W8Params {
    int64_t M, N, K;
    int64_t blocks;  // token blocks of a slice
    int64_t slices;
    const float* scale;  // (M, groups)
    int64_t groups;
    const float* row;  // nullable
    const float* col;  // nullable
    void* dw;
    int64_t ldw;
    int out_type;
    float* work;  // (slices, N, ldp) partial sums
    int64_t ldp;
    int in_work;  // the result goes through work
    int seg;      // token blocks that accumulate in TMEM before the sums leave it
    int dy_blocks, q_blocks;  // tensor maps by column blocks: one box a tile (see w8_launch)
    int* err;
};
struct W8Maps {
    CUtensorMap dy, q;
};

__device__ __forceinline__ void w8_store(void* dw, int64_t at, int out_type, float v) {
    if (out_type == MMB_F32) static_cast<float*>(dw)[at] = v;
    else if (out_type == MMB_BF16) static_cast<__nv_bfloat16*>(dw)[at] = __float2bfloat16_rn(v);
    else static_cast<__half*>(dw)[at] = __float2half_rn(v);
}

// 4 bytes q -> 4 floats q * f.  A byte with its sign bit flipped, q + 128, becomes
// the second byte of the mantissa of 2^15; one fused step then takes 2^15 + 128
// away and multiplies: (2^15 + 128 + q) * f - (2^15 + 128) * f, exact for a power
// of two.
__device__ __forceinline__ void w8_widen4(uint32_t w, float f, float fc, float2& v0, float2& v1) {
    const uint32_t u = w ^ 0x80808080u;
    v0 = ffma2(make_float2(__uint_as_float(__byte_perm(u, 0x47000000u, 0x7404)),
                           __uint_as_float(__byte_perm(u, 0x47000000u, 0x7414))), f2(f), f2(fc));
    v1 = ffma2(make_float2(__uint_as_float(__byte_perm(u, 0x47000000u, 0x7424)),
                           __uint_as_float(__byte_perm(u, 0x47000000u, 0x7434))), f2(f), f2(fc));
}
constexpr float W8_HUGE = 0x1p111f;

template <class D>
__global__ void __launch_bounds__(w8_threads<D>(), 1)
    w8_kernel(const W8Params p, const __grid_constant__ W8Maps maps) {
    using Sm = W8Smem<D>;
    constexpr int RL = D::RL, RC = D::RC, BN = D::BN, BT = D::BT;
    constexpr int AG = D::AG, RA = D::RA, KT = AG * W8_BK;
    constexpr int ACC = D::F32 ? 2 * BN : AG * BN;  // TMEM columns of an accumulator
    constexpr int ROW = AG * BT;                     // place of the row factors behind the scales
    constexpr int CGW = D::CW / D::CG, CT = 32 * CGW;  // a converter group
    constexpr uint32_t IDESC = w8_idesc(BN);
    extern __shared__ float4 w8_smem4[];
    __shared__ uint64_t full[RL], free_l[RL], conv[RC], free_c[RC], acc_full[RA], acc_empty[RA],
        drained;
    __shared__ uint32_t tmem_base_s;
    __shared__ int abort_s;
    volatile int* abort = &abort_s;
    char* smem = reinterpret_cast<char*>(
        (reinterpret_cast<uintptr_t>(w8_smem4) + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    const int64_t kt = (p.K + KT - 1) / KT, nt = (p.N + BN - 1) / BN;
    const int64_t tiles = kt * nt, units = tiles * p.slices;
    const int64_t nblk = (p.M + BT - 1) / BT;
    // unit u: slice, then tile with k fastest: CTAs that run together share tokens
    auto unit_of = [&](int64_t u, int64_t& k0, int64_t& n0, int64_t& b0, int& nb) {
        const int64_t z = u / tiles, t = u % tiles;
        k0 = (t % kt) * KT;
        n0 = (t / kt) * BN;
        b0 = z * p.blocks;
        nb = (int)(min64(nblk, b0 + p.blocks) - b0);
    };
    auto slot_dy = [&](int s) { return smem + s * Sm::LOAD; };
    auto slot_q = [&](int s) { return smem + s * Sm::LOAD + Sm::DY; };
    auto slot_f = [&](int s) {
        return reinterpret_cast<float*>(smem + s * Sm::LOAD + Sm::DY + Sm::Q);
    };
    auto slot_a = [&](int c) { return smem + RL * Sm::LOAD + c * Sm::CONV; };

    if (tid == 0) {
        abort_s = 0;
        for (int s = 0; s < RL; ++s) {
            mbar_init(&full[s], 1 + 32);               // TMA, and the factors of each lane
            mbar_init(&free_l[s], D::PARTS > 1 ? CGW : 1);  // read by the converters / the MMAs
        }
        for (int c = 0; c < RC; ++c) {
            mbar_init(&conv[c], CGW);
            mbar_init(&free_c[c], 1);
        }
        for (int a = 0; a < RA; ++a) {
            mbar_init(&acc_full[a], 1);
            mbar_init(&acc_empty[a], D::EW);
        }
        mbar_init(&drained, 1);
        mbar_fence_init();
    }
    if (warp == 1) tmem_alloc(&tmem_base_s, RA * ACC);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_s;

    if (warp == 0) {
        // ---- producer ----
        if (lane == 0) {
            RingPos<RL> r;
            int64_t j = 0;
            bool ok = true;
            for (int64_t u = blockIdx.x; u < units && ok; u += gridDim.x) {
                int64_t k0, n0, b0;
                int nb;
                unit_of(u, k0, n0, b0, nb);
                const int kx = (int)k0, nx = (int)n0, kg = (int)(k0 / W8_BK), ng = (int)(n0 / 64);
                int m0 = (int)(b0 * BT);
                for (int b = 0; b < nb; ++b, ++j, m0 += BT, r.next()) {
                    uint64_t* bar = &full[r.s];
                    ok = ws_wait(&free_l[r.s], r.ph ^ 1u, abort, p.err);
                    if (!ok) break;
                    mbar_expect_tx(bar, Sm::DY + Sm::Q);
                    if constexpr (D::PARTS > 1) {
                        tma_load_3d(slot_dy(r.s), &maps.dy, nx, m0, 0, bar);
                    } else if (p.dy_blocks) {
                        tma_load_3d(slot_dy(r.s), &maps.dy, 0, m0, ng, bar);
                    } else {
#pragma unroll
                        for (int c = 0; c < BN / 64; ++c)
                            tma_load_3d(slot_dy(r.s) + c * BT * 128, &maps.dy, nx + 64 * c, m0, 0, bar);
                    }
                    if (AG == 1 || p.q_blocks) {
                        tma_load_3d(slot_q(r.s), &maps.q, AG == 1 ? kx : 0, m0, AG == 1 ? 0 : kg, bar);
                    } else {
#pragma unroll
                        for (int g = 0; g < AG; ++g)
                            tma_load_3d(slot_q(r.s) + g * Sm::Q1, &maps.q, kx + g * W8_BK, m0, 0, bar);
                    }
                }
            }
            // copies still in flight land before the CTA leaves
            for (int64_t q = j - RL > 0 ? j - RL : 0; q < j; ++q)
                mbar_wait_polls(&full[q % RL], (uint32_t)((q / RL) & 1), 1 << 16);
        }
    } else if (warp == 2) {
        // ---- the tokens' factors, a token or two a lane, by cp.async ----
        RingPos<RL> r;
        bool ok = true;
        for (int64_t u = blockIdx.x; u < units && ok; u += gridDim.x) {
            int64_t k0, n0, b0;
            int nb;
            unit_of(u, k0, n0, b0, nb);
            const int64_t g0 = k0 / W8_BK;
            int64_t m = b0 * BT + lane;
            const float* sc = p.scale + m * p.groups + g0;
            const int64_t next = 32 * p.groups;
            for (int b = 0; b < nb; ++b, r.next()) {
                ok = __all_sync(0xffffffffu, ws_wait(&free_l[r.s], r.ph ^ 1u, abort, p.err));
                if (!ok) break;
                float* f = slot_f(r.s) + lane;
#pragma unroll
                for (int t = 0; t < BT; t += 32, m += 32, sc += next) {
                    const bool in = m < p.M;
#pragma unroll
                    for (int g = 0; g < AG; ++g) {
                        const bool have = in && (AG == 1 || g0 + g < p.groups);
                        cp_async4(f + g * BT + t, have ? sc + g : p.scale, have);
                    }
                    if (p.row) cp_async4(f + ROW + t, in ? p.row + m : p.row, in);
                }
                cp_async_arrive(&full[r.s]);
            }
        }
        cp_async_commit();
        cp_async_wait<0>();
    } else if (warp == 1) {
        // ---- MMA issuer ----
        if (lane == 0) {
            RingPos<RL> rl;
            RingPos<RC> rc;
            RingPos<RA> ra;
            bool ok = true;
            const uint64_t d0 = smem_desc(smem_u32(smem), BT * 128, 1024, W8_SWZ128);
            const uint32_t lo0 = (uint32_t)d0, dhi = (uint32_t)(d0 >> 32);
            for (int64_t u = blockIdx.x; u < units && ok; u += gridDim.x) {
                int64_t k0, n0, b0;
                int nb;
                unit_of(u, k0, n0, b0, nb);
                int in_seg = 0;
                for (int b = 0; b < nb; ++b, rl.next(), rc.next()) {
                    const int a = ra.s;
                    if (in_seg == 0) {
                        ok = ws_wait(&acc_empty[a], ra.ph ^ 1u, abort, p.err);
                        if (!ok) break;
                        tc_fence_after();
                    }
                    const uint32_t acc = tmem + (uint32_t)(a * ACC);
                    const int s = rl.s, c = rc.s;
                    ok = ws_wait(&conv[c], rc.ph, abort, p.err);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t la = lo0 + (RL * Sm::LOAD + c * Sm::CONV) / 16;
                    const uint32_t lb =
                        D::PARTS > 1 ? la + Sm::A / 16 : lo0 + s * (Sm::LOAD / 16);
                    const uint32_t first = in_seg > 0 ? 1u : 0u;
                    if constexpr (D::F32) {
                        // high and middle parts lie side by side: one MMA of twice the
                        // columns reads the checkpoint once for both
#pragma unroll
                        for (int kk = 0; kk < BT / 16; ++kk) {
                            umma_f16(acc, la + kk * W8_STEP, lb + kk * W8_STEP, dhi,
                                     w8_idesc(2 * BN), kk > 0 ? 1u : first);
                            umma_f16(acc + BN, la + kk * W8_STEP,
                                     lb + 2 * (Sm::P1 / 16) + kk * W8_STEP, dhi, IDESC, 1u);
                        }
                    } else {
#pragma unroll
                        for (int kk = 0; kk < BT / 16; ++kk)
#pragma unroll
                            for (int i = 0; i < D::PARTS; ++i)
#pragma unroll
                                for (int g = 0; g < AG; ++g)
                                    umma_f16(acc + g * BN, la + g * (Sm::A1 / 16) + kk * W8_STEP,
                                             lb + i * (Sm::P1 / 16) + kk * W8_STEP, dhi, IDESC,
                                             kk > 0 || i > 0 ? 1u : first);
                    }
                    if constexpr (D::PARTS == 1) umma_commit(&free_l[s]);
                    umma_commit(&free_c[c]);
                    if (++in_seg == p.seg || b == nb - 1) {
                        umma_commit(&acc_full[a]);
                        ra.next();
                        in_seg = 0;
                    }
                }
            }
            // every MMA this CTA issued has completed before TMEM is freed
            umma_commit(&drained);
            mbar_wait_polls(&drained, 0, 1 << 20);
        }
    } else if (warp < 3 + D::CW) {
        // ---- converters ----
        constexpr int PIECES = BT * W8_BK / 16 / CT;  // 16-byte pieces of q a thread and block
        const int group = (warp - 3) / CGW, ct = (tid - 96) % CT;
        // a piece is 16 columns of a token; 8 neighbouring lanes take the first block's
        // pieces of one token and the second's of its neighbour, so that their stores
        // touch all 8 chunks of a row
        const int piece = ct & 7, blk = piece >> 2, c0 = (piece & 3) * 2;
        const int t0 = 2 * (ct >> 4) + (((ct >> 3) & 1) ^ blk);
        RingPos<RL> rl;
        RingPos<RC> rc;
        RingPos<D::CG> turn;
        bool ok = true;
        for (int64_t u = blockIdx.x; u < units && ok; u += gridDim.x) {
            int64_t k0, n0, b0;
            int nb;
            unit_of(u, k0, n0, b0, nb);
            for (int b = 0; b < nb; ++b, rl.next(), rc.next(), turn.next()) {
                if (turn.s != group) continue;
                const int s = rl.s, cs = rc.s;
                ok = ws_wait(&free_c[cs], rc.ph ^ 1u, abort, p.err) &&
                     ws_wait(&full[s], rl.ph, abort, p.err);
                ok = __all_sync(0xffffffffu, ok);  // a warp leaves together
                if (!ok) break;
                const uint32_t fs = smem_u32(slot_f(s)), qs = smem_u32(slot_q(s)) + piece * 16;
                const uint32_t as = smem_u32(slot_a(cs));
                // every load before the first store, which would hold later loads back
                uint4 w[AG * PIECES];
                float fa[AG * PIECES];
                bool huge = false;
#pragma unroll
                for (int gi = 0; gi < AG * PIECES; ++gi) {
                    const int g = gi / PIECES, t = t0 + gi % PIECES * (CT / 8);
                    w[gi] = lds16(qs + g * Sm::Q1 + t * W8_BK);
                    fa[gi] = lds4f(fs + 4 * (g * BT + t));
                    huge |= fabsf(fa[gi]) >= W8_HUGE;
                }
                const auto widen = [&](float shrink, float grow) {
#pragma unroll
                    for (int gi = 0; gi < AG * PIECES; ++gi) {
                        const int g = gi / PIECES, t = t0 + gi % PIECES * (CT / 8);
                        const float f = fa[gi] * shrink, fc = -32896.f * f;
                        const uint32_t ws[4] = {w[gi].x, w[gi].y, w[gi].z, w[gi].w};
                        uint32_t o[8];
#pragma unroll
                        for (int h = 0; h < 4; ++h) {
                            float2 v0, v1;
                            w8_widen4(ws[h], f, fc, v0, v1);
                            o[2 * h] = w8_pack2(v0.x * grow, v0.y * grow);
                            o[2 * h + 1] = w8_pack2(v1.x * grow, v1.y * grow);
                        }
                        const uint32_t a = as + g * Sm::A1;
                        sts16(a + w8_chunk<BT>(blk, t, c0), make_uint4(o[0], o[1], o[2], o[3]));
                        sts16(a + w8_chunk<BT>(blk, t, c0 + 1), make_uint4(o[4], o[5], o[6], o[7]));
                    }
                };
                // factors of 2^111 and more (values near the type's own limit) go in two
                // steps: 2^15 times them would be an infinity
                if (__any_sync(0xffffffffu, huge)) widen(0x1p-32f, 0x1p32f);
                else widen(1.f, 1.f);
                // dy * row in bf16 parts.  A block with values at fp32's own limit is split a
                // second time, with care
                if constexpr (D::F32) {
                    // high, middle and low: 4 columns of either block of 64 a step (16 lanes
                    // then cover a row of each)
                    const int c = ct & 15;
                    constexpr int STEPS = BT * BN / 8 / CT, AT_ONCE = 4;
                    static_assert(STEPS % AT_ONCE == 0, "whole batches");
                    const uint32_t ds = smem_u32(slot_dy(s)) + c * 16;
                    const auto split = [&](const uint4& x, float r, int t, int h, auto parts) {
                        const uint32_t dst = as + Sm::A + w8_chunk<BT>(h, t, c >> 1) + (c & 1) * 8;
                        const float2 v0 = fmul2(
                            make_float2(__uint_as_float(x.x), __uint_as_float(x.y)), f2(r));
                        const float2 v1 = fmul2(
                            make_float2(__uint_as_float(x.z), __uint_as_float(x.w)), f2(r));
                        uint32_t o0[3], o1[3];
                        parts(v0, o0);
                        parts(v1, o1);
#pragma unroll
                        for (int i = 0; i < 3; ++i) sts8(dst + i * Sm::P1, o0[i], o1[i]);
                    };
                    float top = 0.f;
#pragma unroll
                    for (int i0 = 0; i0 < STEPS; i0 += AT_ONCE) {
                        uint4 x[AT_ONCE][2];
                        float r[AT_ONCE];
#pragma unroll
                        for (int i = 0; i < AT_ONCE; ++i) {
                            const int t = (ct >> 4) + (i0 + i) * (CT / 16);
                            x[i][0] = lds16(ds + t * (BN * 4));
                            x[i][1] = lds16(ds + t * (BN * 4) + 256);
                            r[i] = p.row ? lds4f(fs + 4 * (ROW + t)) : 1.f;
                        }
#pragma unroll
                        for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
                            for (int h = 0; h < 2; ++h)
                                split(x[i][h], r[i], (ct >> 4) + (i0 + i) * (CT / 16), h,
                                      [&](float2 v, uint32_t (&o)[3]) {
                                          top = w8_top(top, v);
                                          w8_parts<3>(v, o);
                                      });
                    }
                    if (__any_sync(0xffffffffu, top >= W8_EDGE)) {
#pragma unroll 1
                        for (int i = 0; i < 2 * STEPS; ++i) {
                            const int t = (ct >> 4) + (i >> 1) * (CT / 16), h = i & 1;
                            split(lds16(ds + t * (BN * 4) + h * 256),
                                  p.row ? lds4f(fs + 4 * (ROW + t)) : 1.f, t, h,
                                  [](float2 v, uint32_t (&o)[3]) { w8_parts_edge<3>(v, o); });
                        }
                    }
                }
                if constexpr (D::PARTS == 2) {
                    // high and low: 8 neighbouring lanes take the 128 bytes of a block of 64
                    // columns of one token
                    const int c = ct & 7;
                    constexpr int ITEMS = BT * (BN / 64), STEPS = ITEMS / (CT / 8), AT_ONCE = 4;
                    static_assert(STEPS % AT_ONCE == 0, "whole batches");
                    const uint32_t ds = smem_u32(slot_dy(s)) + c * 16;
                    const auto load = [&](int i, uint4& x, float& r) {
                        const int item = (ct >> 3) + i * (CT / 8);
                        const int t = item / (BN / 64), h = item % (BN / 64);
                        x = lds16(ds + t * (BN * 2) + h * 128);
                        r = p.row ? lds4f(fs + 4 * (ROW + t)) : 1.f;
                    };
                    const auto split = [&](int i, const uint4& x, float r, auto parts) {
                        const int item = (ct >> 3) + i * (CT / 8);
                        const int t = item / (BN / 64), h = item % (BN / 64);
                        const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
                        uint32_t o[4][2];
#pragma unroll
                        for (int e = 0; e < 4; ++e) parts(fmul2(D::dy2(xs[e]), f2(r)), o[e]);
                        const uint32_t dst = as + Sm::A + w8_chunk<BT>(h, t, c);
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                            sts16(dst + k * Sm::P1, make_uint4(o[0][k], o[1][k], o[2][k], o[3][k]));
                    };
                    float top = 0.f;
#pragma unroll
                    for (int i0 = 0; i0 < STEPS; i0 += AT_ONCE) {
                        uint4 x[AT_ONCE];
                        float r[AT_ONCE];
#pragma unroll
                        for (int i = 0; i < AT_ONCE; ++i) load(i0 + i, x[i], r[i]);
#pragma unroll
                        for (int i = 0; i < AT_ONCE; ++i)
                            split(i0 + i, x[i], r[i], [&](float2 v, uint32_t (&o)[2]) {
                                top = w8_top(top, v);
                                w8_parts<2>(v, o);
                            });
                    }
                    if (__any_sync(0xffffffffu, top >= W8_EDGE)) {
#pragma unroll 1
                        for (int i = 0; i < STEPS; ++i) {
                            uint4 x;
                            float r;
                            load(i, x, r);
                            split(i, x, r,
                                  [](float2 v, uint32_t (&o)[2]) { w8_parts_edge<2>(v, o); });
                        }
                    }
                }
                fence_proxy_async_smem();
                warp_arrive(&conv[cs]);
                if constexpr (D::PARTS > 1) warp_arrive(&free_l[s]);
            }
        }
    } else {
        // ---- epilogue: warp q = warp % 4 reads TMEM lanes (columns k) 32q..32q+31,
        // every 4 warps a share of the columns n ----
        const int q = warp & 3;
        constexpr int COLS = BN / (D::EW / 4);
        const int col0 = ((warp - 3 - D::CW) >> 2) * COLS;
        RingPos<RA> ra;
        bool ok = true;
        for (int64_t u = blockIdx.x; u < units && ok; u += gridDim.x) {
            int64_t k0, n0, b0;
            int nb;
            unit_of(u, k0, n0, b0, nb);
            const int ncols = (int)min64(p.N - n0, BN);
            float* slice = p.in_work ? p.work + ((u / tiles) * p.N + n0) * p.ldp + k0 : nullptr;
            // V columns n0 + c .. of this lane's column k; every segment but the first adds
            // to the sums that this thread left there (in fp32: w8_launch)
            const auto put = [&](int g, int c, auto& v, bool first, bool last) {
                constexpr int V = sizeof(v) / sizeof(v[0]);
                const int kr = g * W8_BK + q * 32 + lane;
                if (k0 + kr >= p.K) return;
                if (!first) {
                    const int64_t ld = slice ? p.ldp : p.ldw;
                    const float* o = slice ? slice + c * p.ldp + kr
                                           : static_cast<const float*>(p.dw) + (n0 + c) * p.ldw + k0 + kr;
#pragma unroll
                    for (int i0 = 0; i0 < V; i0 += 16) {
                        float old[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i, o += ld) old[i] = c + i0 + i < ncols ? *o : 0.f;
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[i0 + i] += old[i];
                    }
                }
                if (slice) {
                    float* w = slice + c * p.ldp + kr;
#pragma unroll
                    for (int i = 0; i < V; ++i, w += p.ldp)
                        if (c + i < ncols) *w = v[i];
                } else {
                    const float cs = p.col && last ? p.col[k0 + kr] : 1.f;
                    int64_t at = (n0 + c) * p.ldw + k0 + kr;
#pragma unroll
                    for (int i = 0; i < V; ++i, at += p.ldw)
                        if (c + i < ncols) w8_store(p.dw, at, p.out_type, v[i] * cs);
                }
            };
            if constexpr (D::F32) {
                float sum[COLS];
#pragma unroll
                for (int i = 0; i < COLS; ++i) sum[i] = 0.f;
                for (int b = 0; b < nb; b += p.seg, ra.next()) {
                    const int a = ra.s;
                    ok = __all_sync(0xffffffffu, ws_wait(&acc_full[a], ra.ph, abort, p.err));
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t trow =
                        tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(a * ACC + col0);
#pragma unroll
                    for (int h = 0; h < 2; ++h)  // the small parts, then the high ones
#pragma unroll
                        for (int c = 0; c < COLS; c += 16) {
                            float r[16];
                            tmem_ld16(trow + (uint32_t)((h ? 0 : BN) + c), r);
#pragma unroll
                            for (int i = 0; i < 16; ++i) sum[c + i] += r[i];
                        }
                    tc_fence_before();
                    warp_arrive(&acc_empty[a]);
                }
                if (!ok) break;
                put(0, col0, sum, true, true);
            } else {
                for (int b = 0; b < nb; b += p.seg, ra.next()) {
                    const int a = ra.s;
                    ok = __all_sync(0xffffffffu, ws_wait(&acc_full[a], ra.ph, abort, p.err));
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t trow = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(a * ACC);
#pragma unroll 1
                    for (int gc = 0; gc < AG * COLS; gc += 32) {
                        const int g = gc / COLS, c = col0 + gc % COLS;
                        float v[32];
                        tmem_ld32(trow + (uint32_t)(g * BN + c), v);
                        put(g, c, v, b == 0, nb - b <= p.seg);
                        __syncwarp();
                    }
                    tc_fence_before();
                    warp_arrive(&acc_empty[a]);
                }
                if (!ok) break;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, RA * ACC);
    }
}

// dw[n, k] = col[k] * sum of the slices' [n, k]: 4 columns a thread (blockDim.x of
// them a block), the slices dealt to blockDim.y groups of threads, always in the
// same order.  Many slices of a small result take 8 groups (37 slices of 512 x 128:
// 6.7 -> 3.6 us), few slices of a large one take 1 (2 of 4096 x 1024: 46 -> 10 us).
constexpr int W8_SUM_NT = 256, W8_SUM_GROUPS = 8;
__global__ void __launch_bounds__(W8_SUM_NT)
    w8_sum_kernel(int64_t N, int64_t K, const float* __restrict__ work, int64_t ldp,
                  int64_t slices, const float* __restrict__ col, void* dw, int64_t ldw,
                  int out_type) {
    __shared__ float4 s[W8_SUM_NT];
    const int qi = threadIdx.x, zi = threadIdx.y, nq = blockDim.x, nz = blockDim.y;
    const int64_t quads = ldp / 4, i = (int64_t)blockIdx.x * nq + qi;
    const bool in = i < N * quads;
    const int64_t n = in ? i / quads : 0, k = in ? (i % quads) * 4 : 0;
    const float* w = work + n * ldp + k;
    float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
    if (in) {
#pragma unroll 4
        for (int64_t z = zi; z < slices; z += nz) {
            const float4 v = *reinterpret_cast<const float4*>(w + z * N * ldp);
            t.x += v.x; t.y += v.y; t.z += v.z; t.w += v.w;
        }
    }
    if (nz > 1) {
        s[zi * nq + qi] = t;
        __syncthreads();
        if (zi) return;
        for (int g = 1; g < nz; ++g) {
            const float4 v = s[g * nq + qi];
            t.x += v.x; t.y += v.y; t.z += v.z; t.w += v.w;
        }
    }
    if (!in) return;
    const float v[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (k + j < K) w8_store(dw, n * ldw + k + j, out_type, col ? v[j] * col[k + j] : v[j]);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
// Slices of the tokens: the count with the least estimated time, a round of
// units costing its token blocks plus a tile's way out, and every slice one
// more write and read of the result.  The costs of blocks and tiles are weights, not
// times: measured with 148 tiles of one slice, a block takes 0.51 us (fp32), 0.54 and
// 0.86 (one part, one and two groups), 0.64 and 0.86 (two parts), a tile's start and way
// out 8, 12 and 20.  With those figures 13 sizes took as long, up to 15 % longer
// (8192 x (2048, 2048) bf16 85 -> 98 us) or 2 % less: rounds overlap, and slices share
// dy in L2, which no cost here knows of.
struct W8Plan {
    int64_t slices, blocks;
    double us;
};
template <class D>
static W8Plan w8_plan(int64_t M, int64_t N, int64_t K) {
    const int64_t nblk = (M + D::BT - 1) / D::BT, kt = D::AG * W8_BK;
    const int64_t tiles = (K + kt - 1) / kt * ((N + D::BN - 1) / D::BN);
    const double block_us = D::F32 ? 0.25 : D::AG == 1 ? 0.45 : 0.60;  // a block of BT tokens
    const double tile_us = 1.0 + D::AG * (D::F32 ? 0.5 : 1.0);
    const double slice_us = 2.0 * (double)N * (double)K * 4.0 / 5e6;
    W8Plan best{1, nblk, 1e30};
    const auto consider = [&](int64_t s) {
        s = s < 1 ? 1 : s > nblk ? nblk : s;
        const int64_t per = (nblk + s - 1) / s;
        s = (nblk + per - 1) / per;  // the slices that this many blocks each make
        const int64_t rounds = (tiles * s + 147) / 148;
        const double t = (double)rounds * ((double)per * block_us + tile_us) +
                         (s > 1 ? 2.0 + (double)s * slice_us : 0.0);
        if (t < best.us) best = {s, per, t};
    };
    for (int64_t r = 1; r <= 4; ++r) consider(148 * r / tiles);  // r full rounds of the SMs
    for (int64_t s = 1; s <= 128; s *= 2) consider(s);
    return best;
}
// 16-bit dy: one group a tile or two, whichever is estimated faster
template <class One, class Two>
static bool w8_two_groups(int64_t M, int64_t N, int64_t K) {
    return w8_plan<Two>(M, N, K).us < w8_plan<One>(M, N, K).us;
}
// Tokens that accumulate in TMEM: its fp32 accumulation truncates, so its error grows
// with their number.
template <class D>
static int w8_seg(int out_type) {
    const int tokens = D::F32 ? W8_SEG_FP32_DY : out_type == MMB_F32 ? W8_SEG_FP32_DW
                                               : W8_SEG_16_DW / D::PARTS;
    return tokens / D::BT;
}
// Several slices, or sums that leave TMEM more than once and have no fp32 result to
// gather in, go through the workspace.
template <class D>
static bool w8_in_work(const W8Plan& plan, int out_type) {
    return plan.slices > 1 || (!D::F32 && out_type != MMB_F32 && plan.blocks > w8_seg<D>(out_type));
}
template <class D>
static int64_t w8_work_slices(int64_t M, int64_t N, int64_t K) {
    const W8Plan plan = w8_plan<D>(M, N, K);
    return w8_in_work<D>(plan, MMB_BF16) ? plan.slices : 0;
}
template <class One, class Two>
static int64_t w8_work_slices(int64_t M, int64_t N, int64_t K) {
    return w8_two_groups<One, Two>(M, N, K) ? w8_work_slices<Two>(M, N, K)
                                            : w8_work_slices<One>(M, N, K);
}
static int64_t w8_pitch(int64_t K) { return (K + 3) / 4 * 4; }

template <class D>
static int w8_launch(W8Params p, const void* dy, int64_t lddy, const int8_t* q, int64_t ldq,
                     cudaStream_t s) {
    const W8Plan plan = w8_plan<D>(p.M, p.N, p.K);
    p.slices = plan.slices;
    p.blocks = plan.blocks;
    p.ldp = w8_pitch(p.K);
    p.seg = w8_seg<D>(p.out_type);
    p.in_work = w8_in_work<D>(plan, p.out_type);
    if (p.in_work && !p.work) return MMB_ERR_WORKSPACE;
    W8Maps maps;
    // dy that is multiplied as it is and a pair of groups as (column in a block, token,
    // block) where their widths are whole blocks: one copy a tile instead of one a block
    p.dy_blocks = D::PARTS == 1 && p.N % 64 == 0;
    p.q_blocks = D::AG > 1 && p.K % W8_BK == 0;
    const bool okd =
        D::PARTS > 1 ? mmb_encode_tile_map(&maps.dy, dy, D::BYTES, p.N, p.M, 1, lddy, lddy * p.M,
                                           D::BN, D::BT, 0)
        : p.dy_blocks
            ? mmb_encode_tile_map(&maps.dy, dy, 2, 64, p.M, p.N / 64, lddy, 64, 64, D::BT, 128,
                                  D::BN / 64)
            : mmb_encode_tile_map(&maps.dy, dy, 2, p.N, p.M, 1, lddy, lddy * p.M, 64, D::BT, 128);
    const bool okq = p.q_blocks ? mmb_encode_tile_map(&maps.q, q, 1, W8_BK, p.M, p.K / W8_BK, ldq,
                                                      W8_BK, W8_BK, D::BT, 0, D::AG)
                                : mmb_encode_tile_map(&maps.q, q, 1, p.K, p.M, 1, ldq, ldq * p.M,
                                                      W8_BK, D::BT, 0);
    if (!okd || !okq) return MMB_ERR_ALIGN;
    static int attr[MMB_MAX_DEVICES] = {};
    const int st = mmb_smem_attr(w8_kernel<D>, W8Smem<D>::BYTES, attr);
    if (st != MMB_OK) return st;
    const int64_t kt = D::AG * W8_BK;
    const int64_t units = (p.K + kt - 1) / kt * ((p.N + D::BN - 1) / D::BN) * p.slices;
    w8_kernel<D><<<(unsigned)min64(units, 148), w8_threads<D>(), W8Smem<D>::BYTES, s>>>(p, maps);
    const int rc = mmb_launch_status();
    if (rc != MMB_OK || !p.in_work) return rc;
    const int64_t quads = p.N * (p.ldp / 4);
    const unsigned groups = p.slices >= 2 * W8_SUM_GROUPS ? W8_SUM_GROUPS : 1;
    const unsigned nq = W8_SUM_NT / groups;
    w8_sum_kernel<<<(unsigned)((quads + nq - 1) / nq), dim3(nq, groups), 0, s>>>(
        p.N, p.K, p.work, p.ldp, p.slices, p.col, p.dw, p.ldw, p.out_type);
    return mmb_launch_status();
}

template <class One, class Two>
static int w8_launch16(const W8Params& p, const void* dy, int64_t lddy, const int8_t* q,
                       int64_t ldq, cudaStream_t s) {
    return w8_two_groups<One, Two>(p.M, p.N, p.K) ? w8_launch<Two>(p, dy, lddy, q, ldq, s)
                                                  : w8_launch<One>(p, dy, lddy, q, ldq, s);
}

}  // namespace mmb

using namespace mmb;

extern "C" size_t mmb_wgrad_ck8_work_floats(int64_t M, int64_t N, int64_t K, int32_t dy_type) {
    if (M <= 0 || N <= 0 || K <= 0 || M > INT32_MAX || N > INT32_MAX || K > INT32_MAX) return 0;
    int64_t slices;
    if (dy_type == MMB_F32) {
        slices = w8_work_slices<W8F32>(M, N, K);
    } else {
        // bf16 and fp16 in two parts share a plan; bf16 without a row factor has its own,
        // and whether there is one is not known here
        slices = w8_work_slices<W8Two<true, 1>, W8Two<true, 2>>(M, N, K);
        if (dy_type == MMB_BF16) {
            const int64_t one = w8_work_slices<W8Half<1>, W8Half<2>>(M, N, K);
            slices = slices > one ? slices : one;
        }
    }
    return (size_t)slices * (size_t)N * (size_t)w8_pitch(K);
}

extern "C" int mmb_wgrad_ck8(int64_t M, int64_t N, int64_t K, int32_t dy_type, const void* dy,
                             int64_t lddy, const int8_t* q, int64_t ldq, const float* scale,
                             const float* row, const float* col, int32_t out_type, void* dw,
                             int64_t ldw, float* work, mmb_stream_t stream) {
    MMB_NVTX("mmb_wgrad_ck8");
    if (M < 0 || N <= 0 || K <= 0 || M > INT32_MAX || N > INT32_MAX || K > INT32_MAX)
        return MMB_ERR_SHAPE;
    const auto known = [](int t) { return t == MMB_F32 || t == MMB_BF16 || t == MMB_F16; };
    if (!known(dy_type) || !known(out_type)) return MMB_ERR_UNSUPPORTED;
    if (!dw) return MMB_ERR_NULL;
    if (ldw < K) return MMB_ERR_SHAPE;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (M == 0) {
        const size_t e = out_type == MMB_F32 ? 4 : 2;
        if (cudaMemset2DAsync(dw, (size_t)ldw * e, 0, (size_t)K * e, (size_t)N, s) != cudaSuccess)
            return mmb_launch_status();
        return MMB_OK;
    }
    if (!dy || !q || !scale) return MMB_ERR_NULL;
    if (lddy < N || ldq < K) return MMB_ERR_SHAPE;
    // TMA: 16-byte aligned bases and row pitches
    const int64_t eb = dy_type == MMB_F32 ? 4 : 2;
    if (((uintptr_t)dy & 15) || ((uintptr_t)q & 15) || (lddy * eb) % 16 || (ldq & 15) ||
        ((uintptr_t)work & 15))
        return MMB_ERR_ALIGN;
    W8Params p{};
    p.M = M; p.N = N; p.K = K;
    p.scale = scale; p.groups = (K + W8_BK - 1) / W8_BK; p.row = row; p.col = col;
    p.dw = dw; p.ldw = ldw; p.out_type = out_type; p.work = work;
    p.err = mmb_device_error_flag();
    if (dy_type == MMB_F32) return w8_launch<W8F32>(p, dy, lddy, q, ldq, s);
    if (dy_type == MMB_F16)
        return w8_launch16<W8Two<false, 1>, W8Two<false, 2>>(p, dy, lddy, q, ldq, s);
    return row ? w8_launch16<W8Two<true, 1>, W8Two<true, 2>>(p, dy, lddy, q, ldq, s)
               : w8_launch16<W8Half<1>, W8Half<2>>(p, dy, lddy, q, ldq, s);
}
