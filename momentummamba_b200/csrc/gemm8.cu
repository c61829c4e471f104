// Product of 8-bit rows on the sm_100a tensor cores (tcgen05 kind::i8):
//
//   out[m, n] = (sum_k xq[m, k] wq[n, k]) * xs[m] * ws[n] (+ bias[n])
//
// x are tokens with a scale each, w a linear's weight with a scale per output
// channel, both K-contiguous.  Products and sums are exact 32-bit integers
// (K <= 131071: K * 128^2 < 2^31); they become fp32 once, are scaled and
// shifted in fp32 and rounded once to the output's type.
//
// Two kernels, both 128-byte K blocks (128 values, 4 MMAs) staged by TMA with
// the 128-byte swizzle, out-of-range rows and columns read as zeros:
//
//  * g8_tile_kernel, for products that fill the GPU: persistent, one CTA per
//    SM, 128 tokens x BN channels, roles in separate warps (producer, MMA
//    issuer, eight epilogue warps) over a ring of K blocks and two TMEM
//    accumulators, so tile t + 1 accumulates while tile t is scaled and stored.
//    B200: 16384 x 8192 x 4096, bf16 out: 376 us, 2.92e15 operations/s, 1.78 times
//    the measured bf16 rate; bound by the tensor cores under the power cap (440 us
//    back to back).  76800 x 1024 x 256, fp32 out: 57-63 us, 5.3-5.9 TB/s; bound by
//    writing 315 MB (48 us alone).  Stores of 32 bytes a lane straight from registers
//    took 92 us there (32 lines a store), boxes of 128-byte rows by TMA 63.
//  * g8_split_kernel, for few tokens (a decoding step), where streaming the
//    weights is all there is to do: the weights are the MMA's 128-row operand
//    and MT tokens its columns, K is cut across the CTAs of a cluster, and the
//    cluster adds its partial sums through distributed shared memory (integers:
//    the order does not matter).  B200: one token 4096 x 1024 4.6 us, 48 tokens
//    2048 x 4096 7.1 us, 8 tokens 8192 x 8192 16 us (10 at the copy rate); bound by
//    the latency of a launch, one trip to memory and the cluster's two barriers
//    (about 4.5 us), then by HBM.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "tc_common.cuh"

namespace mmb {

constexpr int G8_BK = 128;  // bytes (= values) of K per block
constexpr int G8_BM = 128;
constexpr uint32_t G8_SWZ128 = 2;  // descriptor mode: 128-byte swizzle, K-major

// 8-bit signed x 8-bit signed -> 32-bit integers, M = 128, N = n
__host__ __device__ constexpr uint32_t i8_idesc(int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void umma_i8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc,
                                        uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// K-major rows of 128 bytes, 8-row groups 1024 bytes apart; step kk is 32 bytes on
__device__ __forceinline__ uint64_t g8_desc(uint32_t saddr, int kk) {
    return smem_desc(saddr + kk * 32, 16, 1024, G8_SWZ128);
}

struct G8Params {
    int64_t M, N, K;
    const float* xs;
    const float* ws;
    const float* bias;  // nullable
    void* out;
    int64_t ldo;
    int tma_out;  // out goes through TMA boxes (16-byte aligned rows)
    int* err;
};
struct G8Maps {
    CUtensorMap x, w, out;
};

template <int OT>
struct G8Out;
template <>
struct G8Out<MMB_F32> {
    using T = float;
    static __device__ __forceinline__ T from_f(float v) { return v; }
};
template <>
struct G8Out<MMB_BF16> {
    using T = __nv_bfloat16;
    static __device__ __forceinline__ T from_f(float v) { return __float2bfloat16_rn(v); }
    static __device__ __forceinline__ uint32_t pack2(float a, float b) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&t);
    }
};
template <>
struct G8Out<MMB_F16> {
    using T = __half;
    static __device__ __forceinline__ T from_f(float v) { return __float2half_rn(v); }
    static __device__ __forceinline__ uint32_t pack2(float a, float b) {
        const __half2 t = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&t);
    }
};

__device__ __forceinline__ void tma_store_box(const CUtensorMap* map, const void* src, int c0,
                                              int c1) {
    asm volatile(
        "cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group"
        " [%0, {%1, %2, %3}], [%4];" ::"l"(reinterpret_cast<uint64_t>(map)),
        "r"(c0), "r"(c1), "r"(0), "r"(smem_u32(src))
        : "memory");
}

// ---------------------------------------------------------------------------
// tiles
// ---------------------------------------------------------------------------
constexpr int G8_EW = 8;  // epilogue warps: two per TMEM lane quarter, half of the columns each
constexpr int G8_NT = 32 * (2 + G8_EW);
constexpr int G8_GROUP_M = 16;  // tiles of a group share their weights' panels in L2
template <int BN>
__host__ __device__ constexpr int g8_ring() { return BN == 256 ? 4 : 6; }
template <int BN>
struct G8Smem {
    static constexpr int A = G8_BM * G8_BK, B = BN * G8_BK, SLOT = A + B;
    static constexpr int EPI = G8_EW * 4096;  // a 4 KB box per epilogue warp
    static constexpr size_t BYTES = (size_t)g8_ring<BN>() * SLOT + EPI;
};

template <int BN, int OT>
__global__ void __launch_bounds__(G8_NT, 1)
    g8_tile_kernel(const G8Params p, const __grid_constant__ G8Maps maps) {
    using Sm = G8Smem<BN>;
    using O = G8Out<OT>;
    using T = typename O::T;
    constexpr int R = g8_ring<BN>();
    constexpr uint32_t IDESC = i8_idesc(BN);
    // 1024-byte aligned: no room to round up (227 KB with the static part)
    extern __shared__ __align__(1024) char g8_smem[];
    __shared__ uint64_t full[R], empty[R], acc_full[2], acc_empty[2], drained;
    __shared__ float4 chan4[2][BN / 4];  // a tile's channel scales and biases
    __shared__ uint32_t tmem_base_s;
    __shared__ int abort_s;
    float(*chan)[BN] = reinterpret_cast<float(*)[BN]>(chan4);
    volatile int* abort = &abort_s;
    char* smem = g8_smem;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (smem_u32(smem) & 1023u) {
        if (tid == 0 && p.err) atomicOr(p.err, 1);
        return;
    }

    const int64_t mt = (p.M + G8_BM - 1) / G8_BM, nt = (p.N + BN - 1) / BN;
    const int64_t ntiles = mt * nt;
    const int nk = (int)((p.K + G8_BK - 1) / G8_BK);
    // tile t: groups of 16 token tiles, within them m fastest
    auto tile_of = [&](int64_t t, int64_t& m0, int64_t& n0) {
        const int64_t g = t / (G8_GROUP_M * nt), r = t % (G8_GROUP_M * nt);
        const int64_t gm = min64(G8_GROUP_M, mt - g * G8_GROUP_M);
        m0 = (g * G8_GROUP_M + r % gm) * G8_BM;
        n0 = (r / gm) * BN;
    };

    if (tid == 0) {
        abort_s = 0;
        for (int s = 0; s < R; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&acc_full[a], 1);
            mbar_init(&acc_empty[a], G8_EW);
        }
        mbar_init(&drained, 1);
        mbar_fence_init();
    }
    if (warp == 1) tmem_alloc(&tmem_base_s, 2 * BN);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_s;

    if (warp == 0) {
        // ---- producer ----
        if (lane == 0) {
            RingPos<R> r;
            int64_t j = 0;
            bool ok = true;
            for (int64_t t = blockIdx.x; t < ntiles && ok; t += gridDim.x) {
                int64_t m0, n0;
                tile_of(t, m0, n0);
                for (int k = 0; k < nk; ++k, ++j, r.next()) {
                    ok = ws_wait(&empty[r.s], r.ph ^ 1u, abort, p.err);
                    if (!ok) break;
                    char* slot = smem + r.s * Sm::SLOT;
                    mbar_expect_tx(&full[r.s], Sm::SLOT);
                    tma_load_3d(slot, &maps.x, k * G8_BK, (int)m0, 0, &full[r.s]);
                    tma_load_3d(slot + Sm::A, &maps.w, k * G8_BK, (int)n0, 0, &full[r.s]);
                }
            }
            // copies still in flight land before the CTA leaves
            for (int64_t q = j - R > 0 ? j - R : 0; q < j; ++q)
                mbar_wait_polls(&full[q % R], (uint32_t)((q / R) & 1), 1 << 16);
        }
    } else if (warp == 1) {
        // ---- MMA issuer ----
        if (lane == 0) {
            RingPos<R> r;
            RingPos<2> ra;
            bool ok = true;
            for (int64_t t = blockIdx.x; t < ntiles && ok; t += gridDim.x, ra.next()) {
                ok = ws_wait(&acc_empty[ra.s], ra.ph ^ 1u, abort, p.err);
                if (!ok) break;
                tc_fence_after();
                const uint32_t acc = tmem + (uint32_t)(ra.s * BN);
                for (int k = 0; k < nk; ++k, r.next()) {
                    ok = ws_wait(&full[r.s], r.ph, abort, p.err);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t sa = smem_u32(smem + r.s * Sm::SLOT);
#pragma unroll
                    for (int kk = 0; kk < G8_BK / 32; ++kk)
                        umma_i8(acc, g8_desc(sa, kk), g8_desc(sa + Sm::A, kk), IDESC,
                                (k > 0 || kk > 0) ? 1u : 0u);
                    umma_commit(&empty[r.s]);
                }
                if (ok) umma_commit(&acc_full[ra.s]);
            }
            // every MMA this CTA issued has completed before TMEM is freed
            umma_commit(&drained);
            mbar_wait_polls(&drained, 0, 1 << 20);
        }
    } else {
        // ---- epilogue: warp q = warp % 4 reads TMEM lanes (tokens) 32q..32q+31; 32
        // columns at a time go through a box in shared memory to a TMA store.  The scales
        // and the bias of a tile are loaded one tile ahead, the channels' through shared
        // memory ----
        const int q = warp & 3, half = (warp - 2) >> 2, et = tid - 64;
        constexpr int PER = BN / 2;  // columns of a warp
        char* box = smem + R * Sm::SLOT + (warp - 2) * 4096;
        RingPos<2> ra;
        int64_t m0, n0;
        float sx = 0.f, wn = 0.f, bn = 0.f;
        const auto ahead = [&](int64_t t) {
            if (t >= ntiles) return;
            tile_of(t, m0, n0);
            const int64_t m = m0 + q * 32 + lane, n = n0 + et;
            sx = m < p.M ? p.xs[m] : 0.f;
            if (et < BN && n < p.N) {
                wn = p.ws[n];
                if (p.bias) bn = p.bias[n];
            }
        };
        ahead(blockIdx.x);
        for (int64_t t = blockIdx.x; t < ntiles; t += gridDim.x, ra.next()) {
            const int64_t m = m0 + q * 32 + lane, nt0 = n0;
            const int ncols = (int)min64(p.N - n0, BN);
            const float sm = sx;
            // the sums are there, and every warp is done with the channels' values of the
            // tile before; a wait that gave up ends the role for all of its warps at once
            if (!bar_and<1, 32 * G8_EW>(ws_wait(&acc_full[ra.s], ra.ph, abort, p.err))) break;
            tc_fence_after();
            if (et < BN) {
                chan[0][et] = wn;
                chan[1][et] = bn;
            }
            ahead(t + gridDim.x);
            asm volatile("bar.sync 1, %0;" ::"n"(32 * G8_EW) : "memory");
            const uint32_t trow =
                tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(ra.s * BN + half * PER);
            uint32_t r[2][32];
            tmem_ld32_issue(trow, r[0]);
            tmem_wait32(r[0]);
#pragma unroll
            for (int c = 0; c < PER; c += 32) {
                const int cur = (c >> 5) & 1, col = half * PER + c;
                if (c + 32 < PER) tmem_ld32_issue(trow + (uint32_t)(c + 32), r[cur ^ 1]);
                if (col < ncols) {
                    float v[32];
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        const float4 w4 = *reinterpret_cast<const float4*>(&chan[0][col + j]);
                        v[j] = (float)(int)r[cur][j] * sm * w4.x;
                        v[j + 1] = (float)(int)r[cur][j + 1] * sm * w4.y;
                        v[j + 2] = (float)(int)r[cur][j + 2] * sm * w4.z;
                        v[j + 3] = (float)(int)r[cur][j + 3] * sm * w4.w;
                    }
                    if (p.bias) {
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            const float4 b4 = *reinterpret_cast<const float4*>(&chan[1][col + j]);
                            v[j] += b4.x; v[j + 1] += b4.y; v[j + 2] += b4.z; v[j + 3] += b4.w;
                        }
                    }
                    if (p.tma_out) {
                        // 32 tokens x 128 bytes a box: 32 fp32 columns, or two chunks of 16-bit ones
                        constexpr bool WIDE = OT == MMB_F32;
                        const int part = WIDE ? 0 : cur;
                        if (part == 0) {
                            if (lane == 0) bulk_wait_read<0>();  // the box before has left
                            __syncwarp();
                        }
                        uint4* row = reinterpret_cast<uint4*>(box + lane * 128);
                        if constexpr (WIDE) {
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                row[j ^ (lane & 7)] = make_uint4(
                                    __float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]),
                                    __float_as_uint(v[4 * j + 2]), __float_as_uint(v[4 * j + 3]));
                        } else {
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                row[(part * 4 + j) ^ (lane & 7)] = make_uint4(
                                    O::pack2(v[8 * j], v[8 * j + 1]),
                                    O::pack2(v[8 * j + 2], v[8 * j + 3]),
                                    O::pack2(v[8 * j + 4], v[8 * j + 5]),
                                    O::pack2(v[8 * j + 6], v[8 * j + 7]));
                        }
                        if (WIDE || part == 1 || col + 32 >= ncols) {
                            fence_proxy_async_smem();
                            __syncwarp();
                            if (lane == 0) {
                                tma_store_box(&maps.out, box, (int)nt0 + col - (part ? 32 : 0),
                                              (int)m - lane);
                                bulk_commit();
                            }
                        }
                    } else {
                        // rows of any alignment: through the box, then a token at a time
                        // with a column a lane (a token a lane took 32 sectors a store)
                        uint4* row = reinterpret_cast<uint4*>(box + lane * 128);
                        __syncwarp();
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            row[j ^ (lane & 7)] = make_uint4(
                                __float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]),
                                __float_as_uint(v[4 * j + 2]), __float_as_uint(v[4 * j + 3]));
                        __syncwarp();
                        const int rows = (int)min64(p.M - (m - lane), 32);
                        T* o = static_cast<T*>(p.out) + (m - lane) * p.ldo + nt0 + col + lane;
                        const float* b = reinterpret_cast<const float*>(box);
                        if (col + lane < ncols)
#pragma unroll 8
                            for (int t = 0; t < rows; ++t, o += p.ldo)
                                *o = O::from_f(b[t * 32 + (((lane >> 2) ^ (t & 7)) << 2) + (lane & 3)]);
                    }
                }
                __syncwarp();
                if (c + 32 < PER) tmem_wait32(r[cur ^ 1]);
            }
            tc_fence_before();
            warp_arrive(&acc_empty[ra.s]);
        }
        if (lane == 0) bulk_wait_read<0>();
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 2 * BN);
    }
}

// ---------------------------------------------------------------------------
// few tokens: weights stream once, K split across a cluster
// ---------------------------------------------------------------------------
constexpr int G8S_NT = 128;
constexpr int G8S_MAX_SPLIT = 8;
// Two CTAs share an SM (at most 108 KB each): a cluster of 8 then needs 4 SMs of a
// GPC, where 8 whole ones often are not free at once (48 x 2048 x 4096: 16 clusters
// of 8 ran in two waves, 12.5 us, of 4 in one, 8.1 us).
template <int MT>
__host__ __device__ constexpr int g8s_ring() { return MT == 16 ? 6 : MT == 32 ? 5 : MT == 64 ? 4 : 3; }
template <int MT>
struct G8SSmem {
    static constexpr int W = 128 * G8_BK, X = MT * G8_BK, SLOT = W + X;
    static constexpr int RING = g8s_ring<MT>() * SLOT;  // >= the MT x 128 partial sums
    static constexpr size_t BYTES = (size_t)RING + 1024;
    static_assert(RING >= MT * 128 * 4, "the ring's space holds the partial sums");
};
__device__ __forceinline__ void cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\t"
                 "barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// 4 values from another CTA of the cluster (volatile: the loads stay between the
// cluster barriers, but nothing waits for one before the next is issued)
__device__ __forceinline__ int4 ld_cluster4(uint32_t saddr, uint32_t rank) {
    int4 v;
    asm volatile("{\n\t.reg .b32 a;\n\t"
                 "mapa.shared::cluster.u32 a, %4, %5;\n\t"
                 "ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [a];\n\t}"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(saddr), "r"(rank));
    return v;
}

// grid (splits, channel tiles, token tiles), cluster (splits, 1, 1)
template <int MT, int OT>
__global__ void __launch_bounds__(G8S_NT, 2)
    g8_split_kernel(const G8Params p, const __grid_constant__ G8Maps maps) {
    using Sm = G8SSmem<MT>;
    using O = G8Out<OT>;
    constexpr int R = g8s_ring<MT>();
    constexpr int TC = MT < 32 ? 32 : MT;  // TMEM columns
    extern __shared__ float4 g8_smem4[];
    __shared__ uint64_t full[R], empty[R], done;
    __shared__ uint32_t tmem_base_s;
    __shared__ int abort_s;
    volatile int* abort = &abort_s;
    char* smem = reinterpret_cast<char*>(
        (reinterpret_cast<uintptr_t>(g8_smem4) + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, warp = tid >> 5;
    const int splits = gridDim.x, rank = blockIdx.x;
    const int64_t n0 = (int64_t)blockIdx.y * 128, m0 = (int64_t)blockIdx.z * MT;
    const int nkb = (int)((p.K + G8_BK - 1) / G8_BK);
    const int per = (nkb + splits - 1) / splits;
    const int kb = rank * per, ke = kb + per < nkb ? kb + per : nkb;
    const int nk = ke > kb ? ke - kb : 0;
    const int active = (nkb + per - 1) / per;  // ranks that have K blocks

    const auto load = [&](int j) {
        char* slot = smem + (j % R) * Sm::SLOT;
        uint64_t* bar = &full[j % R];
        mbar_expect_tx(bar, Sm::SLOT);
        tma_load_3d(slot, &maps.w, (kb + j) * G8_BK, (int)n0, 0, bar);
        tma_load_3d(slot + Sm::W, &maps.x, (kb + j) * G8_BK, (int)m0, 0, bar);
    };
    if (tid == 0) {
        abort_s = 0;
        for (int s = 0; s < R; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(&done, 1);
        mbar_fence_init();
        // the first loads need nothing but the barriers
        for (int j = 0; j < nk && j < R; ++j) load(j);
    }
    if (warp == 1) tmem_alloc(&tmem_base_s, TC);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_s;

    if (tid == 0) {
        int j = nk < R ? nk : R;
        for (; j < nk; ++j) {
            if (!ws_wait(&empty[j % R], (uint32_t)(((j / R) - 1) & 1), abort, p.err)) break;
            load(j);
        }
        for (int q = j - R > 0 ? j - R : 0; q < j; ++q)
            mbar_wait_polls(&full[q % R], (uint32_t)((q / R) & 1), 1 << 16);
    } else if (tid == 32) {
        bool ok = true;
        for (int j = 0; j < nk; ++j) {
            const int s = j % R;
            ok = ws_wait(&full[s], (uint32_t)((j / R) & 1), abort, p.err);
            if (!ok) break;
            tc_fence_after();
            const uint32_t sw = smem_u32(smem + s * Sm::SLOT);
#pragma unroll
            for (int kk = 0; kk < G8_BK / 32; ++kk)
                umma_i8(tmem, g8_desc(sw, kk), g8_desc(sw + Sm::W, kk), i8_idesc(MT),
                        (j > 0 || kk > 0) ? 1u : 0u);
            umma_commit(&empty[s]);
        }
        umma_commit(&done);
        if (!mbar_wait_polls(&done, 0, 1 << 20)) {
            *abort = 1;
            if (p.err) atomicOr(p.err, 1);
        }
    }
    __syncthreads();  // every copy has landed and every MMA is done (or the call has failed)
    tc_fence_after();

    // partial sums, token-major: part[j][channel]
    int* part = reinterpret_cast<int*>(smem);
    const int ch = tid;  // TMEM lane = channel of the tile
    if (nk > 0) {
#pragma unroll
        for (int c = 0; c < TC; c += 32) {
            uint32_t r[32];
            tmem_ld32_issue(tmem + ((uint32_t)(warp * 32) << 16) + (uint32_t)c, r);
            tmem_wait32(r);
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (c + j < MT) part[(c + j) * 128 + ch] = (int)r[j];
        }
    }
    tc_fence_before();
    if (splits > 1) cluster_sync();
    else __syncthreads();
    // each rank finishes its share of the tokens, 4 channels a thread
    const int share = (MT + splits - 1 - rank) / splits;
    for (int i = tid; i < share * 32; i += G8S_NT) {
        const int j = (i >> 5) * splits + rank, c = (i & 31) * 4;
        const int64_t m = m0 + j, n = n0 + c;
        if (m >= p.M || n >= p.N) continue;
        int4 t = make_int4(0, 0, 0, 0);
        if (splits == 1) {
            t = *reinterpret_cast<const int4*>(part + j * 128 + c);
        } else {
            const uint32_t a = smem_u32(part + j * 128 + c);
            int4 v[G8S_MAX_SPLIT];
#pragma unroll
            for (int r = 0; r < G8S_MAX_SPLIT; ++r)
                v[r] = r < active ? ld_cluster4(a, (uint32_t)r) : make_int4(0, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < G8S_MAX_SPLIT; ++r) {
                t.x += v[r].x; t.y += v[r].y; t.z += v[r].z; t.w += v[r].w;
            }
        }
        const float sx = p.xs[m];
        const int acc[4] = {t.x, t.y, t.z, t.w};
        typename O::T* o = static_cast<typename O::T*>(p.out) + m * p.ldo + n;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (n + e >= p.N) break;
            float v = (float)acc[e] * sx * p.ws[n + e];
            if (p.bias) v += p.bias[n + e];
            o[e] = O::from_f(v);
        }
    }
    if (splits > 1) cluster_sync();  // no CTA leaves while its sums are being read
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, TC);
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
template <int BN, int OT>
static int g8_tile_launch(const G8Params& p0, const int8_t* x, int64_t ldx, const int8_t* w,
                          int64_t ldw, cudaStream_t s) {
    G8Params p = p0;
    G8Maps maps;
    if (!mmb_encode_tile_map(&maps.x, x, 1, p.K, p.M, 1, ldx, ldx * p.M, G8_BK, G8_BM, 128) ||
        !mmb_encode_tile_map(&maps.w, w, 1, p.K, p.N, 1, ldw, ldw * p.N, G8_BK, BN, 128))
        return MMB_ERR_ALIGN;
    constexpr int OB = OT == MMB_F32 ? 4 : 2;
    p.tma_out = ((uintptr_t)p.out & 15) == 0 && (p.ldo * OB) % 16 == 0 &&
                mmb_encode_tile_map(&maps.out, p.out, OB, p.N, p.M, 1, p.ldo, p.ldo * p.M,
                                    128 / OB, 32, 128);
    static int attr[MMB_MAX_DEVICES] = {};
    const int st = mmb_smem_attr(g8_tile_kernel<BN, OT>, G8Smem<BN>::BYTES, attr);
    if (st != MMB_OK) return st;
    const int64_t tiles = (p.M + G8_BM - 1) / G8_BM * ((p.N + BN - 1) / BN);
    const unsigned grid = (unsigned)min64(tiles, 148);
    g8_tile_kernel<BN, OT><<<grid, G8_NT, G8Smem<BN>::BYTES, s>>>(p, maps);
    return mmb_launch_status();
}

template <int MT, int OT>
static int g8_split_launch(const G8Params& p, const int8_t* x, int64_t ldx, const int8_t* w,
                           int64_t ldw, cudaStream_t s) {
    G8Maps maps;
    if (!mmb_encode_tile_map(&maps.x, x, 1, p.K, p.M, 1, ldx, ldx * p.M, G8_BK, MT, 128) ||
        !mmb_encode_tile_map(&maps.w, w, 1, p.K, p.N, 1, ldw, ldw * p.N, G8_BK, 128, 128))
        return MMB_ERR_ALIGN;
    static int attr[MMB_MAX_DEVICES] = {};
    const int st = mmb_smem_attr(g8_split_kernel<MT, OT>, G8SSmem<MT>::BYTES, attr);
    if (st != MMB_OK) return st;
    const int64_t nt = (p.N + 127) / 128, mt = (p.M + MT - 1) / MT;
    const int nkb = (int)((p.K + G8_BK - 1) / G8_BK);
    // as many K slices as fit two CTAs an SM, at least two K blocks each (one token,
    // 4096 x 1024: 8 slices of one block 5.5 us, 4 of two 4.6 us)
    int splits = 1;
    while (splits < G8S_MAX_SPLIT && splits * 4 <= nkb && nt * mt * splits * 2 <= 2 * 148)
        splits *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)splits, (unsigned)nt, (unsigned)mt);
    cfg.blockDim = dim3(G8S_NT);
    cfg.dynamicSmemBytes = G8SSmem<MT>::BYTES;
    cfg.stream = s;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = (unsigned)splits;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, g8_split_kernel<MT, OT>, p, maps);
    if (e != cudaSuccess) {
        mmb_record_cuda_error(e);
        cudaGetLastError();
        return MMB_ERR_LAUNCH;
    }
    return mmb_launch_status();
}

template <int OT>
static int g8_dispatch(const G8Params& p, const int8_t* x, int64_t ldx, const int8_t* w,
                       int64_t ldw, cudaStream_t s) {
    const int64_t nt = (p.N + 127) / 128;
    // 128 x 128 tiles that would leave half of the SMs idle: split K instead
    if ((p.M + 127) / 128 * nt <= 74 && nt <= 65535) {
        if (p.M <= 16) return g8_split_launch<16, OT>(p, x, ldx, w, ldw, s);
        if (p.M <= 32) return g8_split_launch<32, OT>(p, x, ldx, w, ldw, s);
        if (p.M <= 64) return g8_split_launch<64, OT>(p, x, ldx, w, ldw, s);
        return g8_split_launch<128, OT>(p, x, ldx, w, ldw, s);
    }
    // 256 channels a tile once that still gives every SM one
    if ((p.M + 127) / 128 * ((p.N + 255) / 256) >= 148)
        return g8_tile_launch<256, OT>(p, x, ldx, w, ldw, s);
    return g8_tile_launch<128, OT>(p, x, ldx, w, ldw, s);
}

}  // namespace mmb

using namespace mmb;

extern "C" int mmb_gemm_q8(int64_t M, int64_t N, int64_t K, const int8_t* x, int64_t ldx,
                           const float* xs, const int8_t* w, int64_t ldw, const float* ws,
                           const float* bias, int32_t out_type, void* out, int64_t ldo,
                           mmb_stream_t stream) {
    MMB_NVTX("mmb_gemm_q8");
    if (M < 0 || N <= 0 || K <= 0 || M > INT32_MAX || N > INT32_MAX || K > 131071)
        return MMB_ERR_SHAPE;
    if (out_type != MMB_F32 && out_type != MMB_BF16 && out_type != MMB_F16)
        return MMB_ERR_UNSUPPORTED;
    if (M == 0) return MMB_OK;
    if (!x || !xs || !w || !ws || !out) return MMB_ERR_NULL;
    if (ldx < K || ldw < K || ldo < N) return MMB_ERR_SHAPE;
    // TMA: 16-byte aligned bases and row pitches
    if (((uintptr_t)x & 15) || ((uintptr_t)w & 15) || (ldx & 15) || (ldw & 15)) return MMB_ERR_ALIGN;
    G8Params p{};
    p.M = M; p.N = N; p.K = K;
    p.xs = xs; p.ws = ws; p.bias = bias; p.out = out; p.ldo = ldo;
    p.err = mmb_device_error_flag();
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (out_type == MMB_F32) return g8_dispatch<MMB_F32>(p, x, ldx, w, ldw, s);
    if (out_type == MMB_BF16) return g8_dispatch<MMB_BF16>(p, x, ldx, w, ldw, s);
    return g8_dispatch<MMB_F16>(p, x, ldx, w, ldw, s);
}
