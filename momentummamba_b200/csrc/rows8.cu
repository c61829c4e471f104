// Row kernels of the 8-bit path, for sm_100a.
//
//  * 8-bit rows (serving): h = x + residual, v = h * weight, and
//        q = rint(v * 127 / max|v|),   scale = max|v| * rstd / 127,
//    so the root-mean-square norm h * rstd * weight stands as q * scale.  rstd
//    is a factor of the whole row: it cancels in q and only the scale holds
//    it, which is why one pass over the row in registers is enough, and why q
//    does not depend on the order in which the squares are summed.
//  * 8-bit checkpoints (training): h is kept in groups of 128 columns, each
//    with the smallest power of two s (at least 2^-100) with max|h| <= 127 s:
//        q = rint(h / s),   kept value q * s
//    (|q| <= 63 where 64 s is beyond h's type, so that it stays finite there: s =
//    2^122, or 2^10 where h is finite fp16).
//    A power of two makes h / s exact, so what is kept is the same on every
//    run, and q * s is exact in bf16 and tf32, which the weight gradient
//    multiplies it in.  The norm h * rstd * weight goes out beside it in the
//    type asked for.
//  * the norm's backward from the checkpoint: with z = kept * rstd,
//        g = dn * weight,   dx = rstd * (g - z * mean(g z)) + dh,
//        dweight = sum over rows of dn * z.
//  * restoring 8-bit rows or checkpoints.
//
// All arithmetic and sums are fp32; only what is stored is rounded, once, to
// its own type.  A row (or group) that holds a NaN or an infinity gets a NaN
// scale: every value it restores to is NaN.
//
// Layout.  A row is held in the registers of W warps, 8 values of a lane per
// chunk, NC chunks of 256 columns per warp (rows of at most 128 columns: two a
// warp).  Aligned rows whose width is a multiple of 8 take 16-byte loads (a lane's
// 8 values are neighbours, half a warp is a group of 128); any other row takes
// single loads, a warp's lanes side by side (a group is 4 values of each of the
// 32 lanes).  All of a row's loads are issued before the first is used.
//
// Everything here is bound by HBM: each value is read once and written once.
// B200, 65536 x 1024 bf16 (bytes at the measured 6.55 TB/s copy rate beside it):
// 8-bit rows 72 us (72), checkpointed norm 93 (92), its backward with the column
// sums 90 (72: blocks walk rows, and a row's load, reduction and store follow one
// another), restoring 33 (31).  65536 x 1001 fp16, single loads: 101 (70),
// 136 (90), 134 (70); these are bound by the number of accesses.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "mmb_common.cuh"

namespace mmb {

constexpr int R8_GROUP = 128;
constexpr int R8_MAX_WARPS = 16;
constexpr int R8_CHUNK = 256;  // columns of one warp and chunk
constexpr float R8_TINY = 7.888609052210118e-31f;  // 2^-100

// ---------------------------------------------------------------------------
// element types: 8 values of a row in registers
// ---------------------------------------------------------------------------
struct T8F32 {
    using T = float;
    struct Raw { float4 a, b; };
    static __device__ __forceinline__ Raw ldv(const T* p) {
        return {reinterpret_cast<const float4*>(p)[0], reinterpret_cast<const float4*>(p)[1]};
    }
    static __device__ __forceinline__ void unpack(const Raw& r, float (&v)[8]) {
        v[0] = r.a.x; v[1] = r.a.y; v[2] = r.a.z; v[3] = r.a.w;
        v[4] = r.b.x; v[5] = r.b.y; v[6] = r.b.z; v[7] = r.b.w;
    }
    static __device__ __forceinline__ void stv(T* p, const float (&v)[8]) {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
    static __device__ __forceinline__ float to_f(T x) { return x; }
    static __device__ __forceinline__ T from_f(float x) { return x; }
};
struct T8BF16 {
    using T = __nv_bfloat16;
    using Raw = uint4;
    static __device__ __forceinline__ Raw ldv(const T* p) {
        return *reinterpret_cast<const uint4*>(p);
    }
    static __device__ __forceinline__ void unpack(const Raw& r, float (&v)[8]) {
        v[0] = bf16_lo(r.x); v[1] = bf16_hi(r.x); v[2] = bf16_lo(r.y); v[3] = bf16_hi(r.y);
        v[4] = bf16_lo(r.z); v[5] = bf16_hi(r.z); v[6] = bf16_lo(r.w); v[7] = bf16_hi(r.w);
    }
    static __device__ __forceinline__ uint32_t pack2(float a, float b) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&t);
    }
    static __device__ __forceinline__ void stv(T* p, const float (&v)[8]) {
        *reinterpret_cast<uint4*>(p) = make_uint4(pack2(v[0], v[1]), pack2(v[2], v[3]),
                                                  pack2(v[4], v[5]), pack2(v[6], v[7]));
    }
    static __device__ __forceinline__ float to_f(T x) { return __bfloat162float(x); }
    static __device__ __forceinline__ T from_f(float x) { return __float2bfloat16_rn(x); }
};
struct T8F16 {
    using T = __half;
    using Raw = uint4;
    static __device__ __forceinline__ Raw ldv(const T* p) {
        return *reinterpret_cast<const uint4*>(p);
    }
    static __device__ __forceinline__ void unpack2(uint32_t w, float& a, float& b) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
        a = f.x;
        b = f.y;
    }
    static __device__ __forceinline__ void unpack(const Raw& r, float (&v)[8]) {
        unpack2(r.x, v[0], v[1]);
        unpack2(r.y, v[2], v[3]);
        unpack2(r.z, v[4], v[5]);
        unpack2(r.w, v[6], v[7]);
    }
    static __device__ __forceinline__ uint32_t pack2(float a, float b) {
        const __half2 t = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&t);
    }
    static __device__ __forceinline__ void stv(T* p, const float (&v)[8]) {
        *reinterpret_cast<uint4*>(p) = make_uint4(pack2(v[0], v[1]), pack2(v[2], v[3]),
                                                  pack2(v[4], v[5]), pack2(v[6], v[7]));
    }
    static __device__ __forceinline__ float to_f(T x) { return __half2float(x); }
    static __device__ __forceinline__ T from_f(float x) { return __float2half_rn(x); }
};

// Column of value j of this lane in the 256-column chunk at c0.
constexpr __host__ __device__ __forceinline__ int r8_off(int j) {
    return (j >> 2) * R8_GROUP + (j & 3) * 32;
}
template <bool VEC>
__device__ __forceinline__ int64_t r8_col(int64_t c0, int lane, int j) {
    return VEC ? c0 + lane * 8 + j : c0 + r8_off(j) + lane;
}

// 8 values of a row, zeros past its end.  Raw form first, so that all of a
// row's loads are issued before the first is used.
template <class E, bool VEC>
struct R8Load;
template <class E>
struct R8Load<E, true> {
    typename E::Raw r;
    __device__ __forceinline__ void load(const typename E::T* row, int64_t c0, int lane,
                                         int64_t cols) {
        const int64_t c = c0 + lane * 8;
        if (c < cols) r = E::ldv(row + c);
        else r = typename E::Raw{};
    }
    __device__ __forceinline__ void get(float (&v)[8]) const { E::unpack(r, v); }
};
template <class E>
struct R8Load<E, false> {
    typename E::T r[8];
    __device__ __forceinline__ void load(const typename E::T* row, int64_t c0, int lane,
                                         int64_t cols) {
        // whole chunks (all but a row's last) without a comparison a value
        const typename E::T* q = row + c0 + lane;
        const int left = (int)(cols - c0) - lane;
        if (cols - c0 >= R8_CHUNK) {
#pragma unroll
            for (int j = 0; j < 8; ++j) r[j] = q[r8_off(j)];
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) r[j] = r8_off(j) < left ? q[r8_off(j)] : E::from_f(0.f);
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = E::to_f(r[j]);
    }
};
template <class E, bool VEC>
__device__ __forceinline__ void r8_store(typename E::T* row, int64_t c0, int lane, int64_t cols,
                                         const float (&v)[8]) {
    if constexpr (VEC) {
        if (c0 + lane * 8 < cols) E::stv(row + c0 + lane * 8, v);
    } else {
        typename E::T* q = row + c0 + lane;
        const int left = (int)(cols - c0) - lane;
        if (cols - c0 >= R8_CHUNK) {
#pragma unroll
            for (int j = 0; j < 8; ++j) q[r8_off(j)] = E::from_f(v[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (r8_off(j) < left) q[r8_off(j)] = E::from_f(v[j]);
        }
    }
}

// rint(t) for |t| <= 2^21, in the low byte: adding 1.5 * 2^23 leaves the value,
// rounded to nearest even, in the low mantissa bits.
__device__ __forceinline__ uint32_t r8_round(float t) {
    return __float_as_uint(__fadd_rn(t, 12582912.f));
}
__device__ __forceinline__ uint32_t r8_pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
template <bool VEC>
__device__ __forceinline__ void r8_store_q(int8_t* row, int64_t c0, int lane, int64_t cols,
                                           const uint32_t (&b)[8]) {
    if constexpr (VEC) {
        if (c0 + lane * 8 < cols)
            *reinterpret_cast<uint2*>(row + c0 + lane * 8) =
                make_uint2(r8_pack4(b[0], b[1], b[2], b[3]), r8_pack4(b[4], b[5], b[6], b[7]));
    } else {
        int8_t* q = row + c0 + lane;
        const int left = (int)(cols - c0) - lane;
        if (cols - c0 >= R8_CHUNK) {
#pragma unroll
            for (int j = 0; j < 8; ++j) q[r8_off(j)] = (int8_t)b[j];
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (r8_off(j) < left) q[r8_off(j)] = (int8_t)b[j];
        }
    }
}
template <bool VEC>
struct R8LoadQ;
template <>
struct R8LoadQ<true> {
    uint2 r;
    __device__ __forceinline__ void load(const int8_t* row, int64_t c0, int lane, int64_t cols) {
        r = c0 + lane * 8 < cols ? *reinterpret_cast<const uint2*>(row + c0 + lane * 8)
                                 : make_uint2(0u, 0u);
    }
    // byte -> float: the byte (with its sign bit flipped) becomes the low
    // mantissa bits of 2^23, from which 2^23 + 128 is taken away
    __device__ __forceinline__ void get(float (&v)[8]) const {
        const uint32_t a = r.x ^ 0x80808080u, b = r.y ^ 0x80808080u;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = __uint_as_float(__byte_perm(a, 0x4b000000u, 0x7440 + j)) - 8388736.f;
            v[4 + j] = __uint_as_float(__byte_perm(b, 0x4b000000u, 0x7440 + j)) - 8388736.f;
        }
    }
};
template <>
struct R8LoadQ<false> {
    int8_t r[8];
    __device__ __forceinline__ void load(const int8_t* row, int64_t c0, int lane, int64_t cols) {
        const int8_t* q = row + c0 + lane;
        const int left = (int)(cols - c0) - lane;
        if (cols - c0 >= R8_CHUNK) {
#pragma unroll
            for (int j = 0; j < 8; ++j) r[j] = q[r8_off(j)];
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) r[j] = r8_off(j) < left ? q[r8_off(j)] : (int8_t)0;
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)r[j];
    }
};

// max that keeps a NaN
__device__ __forceinline__ float r8_max(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// Sum (and maximum) over the row: LPR lanes, then the row's warps (whose number is
// the block's x extent / 32; blocks of several warps hold one row).
template <int LPR, bool MAX>
__device__ __forceinline__ void r8_row_reduce(float& sum, float& top, float2* part) {
#pragma unroll
    for (int m = LPR / 2; m >= 1; m >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, m);
        if constexpr (MAX) top = r8_max(top, __shfl_xor_sync(0xffffffffu, top, m));
    }
    const int nw = blockDim.x >> 5;
    if (LPR < 32 || nw == 1) return;
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = make_float2(sum, top);
    __syncthreads();
    sum = 0.f;
    top = 0.f;
    for (int w = 0; w < nw; ++w) {
        sum += part[w].x;
        if constexpr (MAX) top = r8_max(top, part[w].y);
    }
}

struct R8Fwd {
    int64_t rows, cols;
    const void* x;
    int64_t xs;
    const void* res;  // nullable
    int64_t rs;
    const float* w;  // nullable
    void* h;         // nullable: the sum, in the residual's type
    int64_t hs;
    void* n;  // nullable: the norm (checkpoints only)
    int64_t ns;
    int nt;  // n's type
    int8_t* q;
    int64_t qs;
    float* scale;  // rows, or rows x groups
    float* rstd;   // nullable
    float eps;
    int norm;  // 0: quantise x as it is
};

// CK: checkpoint form (groups, powers of two); else 8-bit rows.
// LPR: lanes of a row, 16 for rows of at most 128 columns (two rows a warp).
template <class EX, class ER, bool VEC, int NC, int NT, bool CK, int LPR = 32>
__global__ void __launch_bounds__(NT) r8_fwd_kernel(const R8Fwd p) {
    __shared__ float2 part[R8_MAX_WARPS];
    constexpr int RPW = 32 / LPR;
    constexpr bool F16 = std::is_same<EX, T8F16>::value, ER_F16 = std::is_same<ER, T8F16>::value;
    const int lane = threadIdx.x & (LPR - 1), warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    const int64_t first = ((int64_t)blockIdx.x * blockDim.y + threadIdx.y) * RPW;
    if (first >= p.rows) return;  // whole warps; blocks of several warps hold one row
    // a half warp past the end goes through the last row again and stores nothing
    const int64_t at = first + (threadIdx.x & 31) / LPR, row = min64(at, p.rows - 1);
    const int64_t cols = at < p.rows ? p.cols : 0;  // columns that are stored
    const auto col0 = [&](int c) { return (int64_t)(c * nw + warp) * R8_CHUNK; };
    const auto* xr = static_cast<const typename EX::T*>(p.x) + row * p.xs;

    float v[NC][8];
    {
        R8Load<EX, VEC> lx[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) lx[c].load(xr, col0(c), lane, p.cols);
        if (p.res) {
            const auto* rr = static_cast<const typename ER::T*>(p.res) + row * p.rs;
            R8Load<ER, VEC> lr[NC];
#pragma unroll
            for (int c = 0; c < NC; ++c) lr[c].load(rr, col0(c), lane, p.cols);
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                float a[8], b[8];
                lx[c].get(a);
                lr[c].get(b);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[c][j] = a[j] + b[j];
            }
        } else {
#pragma unroll
            for (int c = 0; c < NC; ++c) lx[c].get(v[c]);
        }
    }
    if (p.h) {
        auto* hr = static_cast<typename ER::T*>(p.h) + row * p.hs;
#pragma unroll
        for (int c = 0; c < NC; ++c) r8_store<ER, VEC>(hr, col0(c), lane, cols, v[c]);
    }
    float sum = 0.f, top = 0.f;
    if (p.norm) {
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j) sum = fmaf(v[c][j], v[c][j], sum);
    }
    if constexpr (!CK) {
        if (p.w) {
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                R8Load<T8F32, VEC> lw;
                float w[8];
                lw.load(p.w, col0(c), lane, p.cols);
                lw.get(w);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[c][j] *= w[j];
            }
        }
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j) top = r8_max(top, fabsf(v[c][j]));
    }
    if (p.norm || !CK) r8_row_reduce<LPR, !CK>(sum, top, part);
    const float rstd = p.norm ? __frsqrt_rn(__fdiv_rn(sum, (float)p.cols) + p.eps) : 1.f;
    int8_t* qr = p.q ? p.q + row * p.qs : nullptr;

    if constexpr (!CK) {
        // rows whose largest value is below 2^-100 count as zero (127 / top stays finite).
        // The reciprocal times 127, each rounded: what an array library makes of 127 / top,
        // so that a restatement there lands on the same side of every step
        const float inv =
            top >= R8_TINY && top < INFINITY ? __fmul_rn(__frcp_rn(top), 127.f) : 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            uint32_t b[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) b[j] = r8_round(__fmul_rn(v[c][j], inv));
            r8_store_q<VEC>(qr, col0(c), lane, cols, b);
        }
        // rounded down: 127 scales never exceed the row's largest value, which may
        // be the type's own
        if (lane == 0 && warp == 0 && cols)
            p.scale[row] = top < INFINITY ? __fdiv_rd(top * rstd, 127.f) : NAN;
        return;
    } else {
        if (qr) {
            const int64_t groups = (p.cols + R8_GROUP - 1) / R8_GROUP;
            float* sr = p.scale + row * groups;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                // a lane's values fall into one group (VEC) or into two
                float t[VEC ? 1 : 2];
                if constexpr (VEC) {
                    t[0] = 0.f;
#pragma unroll
                    for (int j = 0; j < 8; ++j) t[0] = r8_max(t[0], fabsf(v[c][j]));
#pragma unroll
                    for (int m = 8; m >= 1; m >>= 1)
                        t[0] = r8_max(t[0], __shfl_xor_sync(0xffffffffu, t[0], m));
                } else {
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        t[g] = 0.f;
#pragma unroll
                        for (int j = 0; j < 4; ++j) t[g] = r8_max(t[g], fabsf(v[c][4 * g + j]));
#pragma unroll
                        for (int m = 16; m >= 1; m >>= 1)
                            t[g] = r8_max(t[g], __shfl_xor_sync(0xffffffffu, t[g], m));
                    }
                }
                uint32_t b[8];
#pragma unroll
                for (int g = 0; g < (VEC ? 1 : 2); ++g) {
                    // t = m 2^e, m in [1, 2): t / 2^(e-6) = 64 m, above 127 when m > 127/64
                    const uint32_t u = __float_as_uint(t[g]);
                    int e = (int)(u >> 23) - 127 - 6 + ((u & 0x7fffffu) > 0x7e0000u ? 1 : 0);
                    e = e < -100 ? -100 : e;
                    const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
                    constexpr int V = VEC ? 8 : 4;
                    float q[V];
#pragma unroll
                    for (int j = 0; j < V; ++j) q[j] = __fmul_rn(v[c][V * g + j], inv);
                    bool edge = e == 122;  // values at the type's own limit: 64 s would be 2^128
                    if constexpr (F16) edge |= e == 10 && t[g] < 65520.f && (ER_F16 || !p.res);
                    if (edge) {
#pragma unroll
                        for (int j = 0; j < V; ++j) q[j] = fminf(fmaxf(q[j], -63.f), 63.f);
                    }
#pragma unroll
                    for (int j = 0; j < V; ++j) b[V * g + j] = r8_round(q[j]);
                    const int64_t gc = col0(c) + (VEC ? (lane >> 4) : g) * R8_GROUP;
                    const bool mine = VEC ? (lane & 15) == 0 : lane == 0;
                    if (mine && gc < cols)
                        sr[gc / R8_GROUP] =
                            t[g] < INFINITY ? __uint_as_float((uint32_t)(127 + e) << 23) : NAN;
                }
                r8_store_q<VEC>(qr, col0(c), lane, cols, b);
            }
        }
        if (p.rstd && lane == 0 && warp == 0 && cols) p.rstd[row] = rstd;
        if (p.n) {
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                float o[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) o[j] = v[c][j] * rstd;
                if (p.w) {
                    R8Load<T8F32, VEC> lw;
                    float w[8];
                    lw.load(p.w, col0(c), lane, p.cols);
                    lw.get(w);
#pragma unroll
                    for (int j = 0; j < 8; ++j) o[j] *= w[j];
                }
                if (p.nt == MMB_F32)
                    r8_store<T8F32, VEC>(static_cast<float*>(p.n) + row * p.ns, col0(c), lane,
                                         cols, o);
                else if (p.nt == MMB_BF16)
                    r8_store<T8BF16, VEC>(static_cast<__nv_bfloat16*>(p.n) + row * p.ns, col0(c),
                                          lane, cols, o);
                else
                    r8_store<T8F16, VEC>(static_cast<__half*>(p.n) + row * p.ns, col0(c), lane,
                                         cols, o);
            }
        }
    }
}

struct R8Bwd {
    int64_t rows, cols;
    const void* dn;
    int64_t dns;
    const void* dh;  // nullable, dx's type
    int64_t dhs;
    const float* w;  // nullable
    const int8_t* q;
    int64_t qs;
    const float* scale;  // rows x groups
    const float* rstd;
    void* dx;
    int64_t dxs;
    float* part;  // gridDim.x x cols partial sums of dweight (null: none wanted)
};

// Blocks walk rows, blockDim.y * U at a time: a warp loads U rows at once (narrow
// rows leave too few bytes in flight otherwise: 32768 x 128 fp32 took 24 us with
// one row a warp).  Each thread keeps its columns' share of dweight in
// registers; at the end a block's rows-in-flight are added up in shared memory
// and the block writes its own line of partial sums, which r8_colsum_kernel adds
// in a fixed order: the result does not depend on timing.
// Blocks of 128 threads run four an SM: 153 registers a thread left three (65536 x
// 1024 bf16: 102 us against 94).  With single loads three run, and are launched:
// without the bound their registers left two (65536 x 501 bf16: 144 us against 95).
template <class EN, class EX, bool VEC, int NC, int U, int NT, int LPR = 32>
__global__ void __launch_bounds__(NT, NT != 128 ? 1 : VEC ? 4 : 3) r8_bwd_kernel(const R8Bwd p) {
    extern __shared__ float r8_acc[];  // blockDim.y x cols, when blockDim.y > 1
    __shared__ float2 part[R8_MAX_WARPS];
    constexpr int RPW = 32 / LPR;
    const int lane = threadIdx.x & (LPR - 1), warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    const int sub = (threadIdx.x & 31) / LPR;  // this half warp's row
    const int64_t groups = (p.cols + R8_GROUP - 1) / R8_GROUP;
    const auto col0 = [&](int c) { return (int64_t)(c * nw + warp) * R8_CHUNK; };
    const int64_t step = (int64_t)gridDim.x * blockDim.y * RPW;
    constexpr int G = VEC ? 1 : 2;  // groups a lane's 8 values fall into
    float acc[NC][8];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[c][j] = 0.f;

    for (int64_t row0 = ((int64_t)blockIdx.x * blockDim.y + threadIdx.y) * RPW; row0 < p.rows;
         row0 += step * U) {
        R8Load<EN, VEC> ln[U][NC];
        R8Load<EX, VEC> lh[U][NC];
        R8LoadQ<VEC> lq[U][NC];
        float s[U][NC][G], rstd[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            // a row past the end loads the last one again and stores nothing
            const int64_t row = min64(row0 + sub + u * step, p.rows - 1);
            const auto* dnr = static_cast<const typename EN::T*>(p.dn) + row * p.dns;
#pragma unroll
            for (int c = 0; c < NC; ++c) ln[u][c].load(dnr, col0(c), lane, p.cols);
            if (p.dh) {
                const auto* dhr = static_cast<const typename EX::T*>(p.dh) + row * p.dhs;
#pragma unroll
                for (int c = 0; c < NC; ++c) lh[u][c].load(dhr, col0(c), lane, p.cols);
            }
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                lq[u][c].load(p.q + row * p.qs, col0(c), lane, p.cols);
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const int64_t gc = col0(c) + (VEC ? (lane >> 4) : g) * R8_GROUP;
                    s[u][c][g] = gc < p.cols ? p.scale[row * groups + gc / R8_GROUP] : 0.f;
                }
            }
            rstd[u] = p.rstd[row];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (row0 + u * step >= p.rows) break;  // the same for a warp, and for a block of one row
            const int64_t row = row0 + sub + u * step;
            const bool live = RPW == 1 || row < p.rows;
            float z[NC][8], g[NC][8], dot = 0.f;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                lq[u][c].get(z[c]);
                ln[u][c].get(g[c]);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    z[c][j] *= s[u][c][VEC ? 0 : j >> 2] * rstd[u];
                    if (live) acc[c][j] = fmaf(g[c][j], z[c][j], acc[c][j]);
                }
                if (p.w) {
                    R8Load<T8F32, VEC> lw;
                    float w[8];
                    lw.load(p.w, col0(c), lane, p.cols);
                    lw.get(w);
#pragma unroll
                    for (int j = 0; j < 8; ++j) g[c][j] *= w[j];
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) dot = fmaf(g[c][j], z[c][j], dot);
            }
            float unused = 0.f;
            r8_row_reduce<LPR, false>(dot, unused, part);
            const float mean = __fdiv_rn(dot, (float)p.cols);
            auto* dxr = static_cast<typename EX::T*>(p.dx) + row * p.dxs;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
#pragma unroll
                for (int j = 0; j < 8; ++j) g[c][j] = rstd[u] * fmaf(-z[c][j], mean, g[c][j]);
                if (p.dh) {
                    float a[8];
                    lh[u][c].get(a);
#pragma unroll
                    for (int j = 0; j < 8; ++j) g[c][j] += a[j];
                }
                if (live) r8_store<EX, VEC>(dxr, col0(c), lane, p.cols, g[c]);
            }
            if (nw > 1) __syncthreads();  // `part` is written again for the next row
        }
    }
    if (!p.part) return;
    if constexpr (RPW == 2) {  // the half warps' rows; both then write the same sums
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[0][j] += __shfl_xor_sync(0xffffffffu, acc[0][j], 16);
    }
    float* out = p.part + (int64_t)blockIdx.x * p.cols;
    if (blockDim.y == 1) {
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int64_t k = r8_col<VEC>(col0(c), lane, j);
                if (k < p.cols) out[k] = acc[c][j];
            }
        return;
    }
    float* mine = r8_acc + (int64_t)threadIdx.y * p.cols;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int64_t k = r8_col<VEC>(col0(c), lane, j);
            if (k < p.cols) mine[k] = acc[c][j];
        }
    __syncthreads();
    for (int64_t k = threadIdx.y * blockDim.x + threadIdx.x; k < p.cols;
         k += blockDim.x * blockDim.y) {
        float t = 0.f;
        for (unsigned r = 0; r < blockDim.y; ++r) t += r8_acc[(int64_t)r * p.cols + k];
        out[k] = t;
    }
}

// out[k] = sum of the lines' column k, in a fixed order
constexpr int R8_SUM_ROWS = 32, R8_SUM_COLS = 32;
__global__ void __launch_bounds__(R8_SUM_COLS* R8_SUM_ROWS)
    r8_colsum_kernel(const float* __restrict__ part, int lines, int64_t cols,
                     float* __restrict__ out) {
    __shared__ float s[R8_SUM_ROWS][R8_SUM_COLS];
    const int64_t k = (int64_t)blockIdx.x * R8_SUM_COLS + threadIdx.x;
    float t = 0.f;
    if (k < cols) {
#pragma unroll 8
        for (int l = threadIdx.y; l < lines; l += R8_SUM_ROWS) t += part[(int64_t)l * cols + k];
    }
    s[threadIdx.y][threadIdx.x] = t;
    __syncthreads();
#pragma unroll
    for (int h = R8_SUM_ROWS / 2; h >= 1; h >>= 1) {
        if (threadIdx.y < h) s[threadIdx.y][threadIdx.x] += s[threadIdx.y + h][threadIdx.x];
        __syncthreads();
    }
    if (threadIdx.y == 0 && k < cols) out[k] = s[0][threadIdx.x];
}

// Restored rows: q * scale (one per row, or one per group of 128 columns).  A
// warp takes 256 columns of R8_RROWS rows, all loads first.
constexpr int R8_RROWS = 4;
template <class E, bool VEC>
__global__ void __launch_bounds__(256)
    r8_restore_kernel(int64_t rows, int64_t cols, const int8_t* __restrict__ q, int64_t qs,
                      const float* __restrict__ scale, int64_t groups, void* out, int64_t os) {
    const int lane = threadIdx.x & 31;
    const int64_t c0 = (int64_t)blockIdx.y * R8_CHUNK;
    const int64_t row0 = ((int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)) * R8_RROWS;
    if (row0 >= rows) return;
    constexpr int G = VEC ? 1 : 2;
    R8LoadQ<VEC> lq[R8_RROWS];
    float s[R8_RROWS][G];
#pragma unroll
    for (int i = 0; i < R8_RROWS; ++i) {
        const int64_t row = min64(row0 + i, rows - 1);
        lq[i].load(q + row * qs, c0, lane, cols);
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const int64_t gc = c0 + (VEC ? (lane >> 4) : g) * R8_GROUP;
            s[i][g] = !groups ? scale[row] : gc < cols ? scale[row * groups + gc / R8_GROUP] : 0.f;
        }
    }
#pragma unroll
    for (int i = 0; i < R8_RROWS; ++i) {
        if (row0 + i >= rows) break;
        float v[8];
        lq[i].get(v);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= s[i][VEC ? 0 : j >> 2];
        r8_store<E, VEC>(static_cast<typename E::T*>(out) + (row0 + i) * os, c0, lane, cols, v);
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
// Warps per row, chunks per warp and rows per block.  NC = 0: too wide.
struct R8Shape {
    int warps, nc, rows;  // rows: of a block
    bool half;            // two rows a warp
};
static R8Shape r8_shape(int64_t cols, bool vec) {
    const int64_t chunks = (cols + R8_CHUNK - 1) / R8_CHUNK;
    if (vec && cols <= 128) return {1, 1, 8, true};
    if (chunks <= 1) return {1, 1, 4};
    if (chunks <= 2) return {1, 2, 4};
    // single loads of four chunks take a thread 242 registers in the backward: two
    // warps a row then (65536 x 1001 fp16)
    if (chunks <= 4) return vec ? R8Shape{1, 4, 4} : R8Shape{2, 2, 1};
    // several warps a row: two chunks each as long as 16 warps suffice (four leave
    // a 512-thread block too few registers)
    if (chunks <= 2 * R8_MAX_WARPS) return {(int)((chunks + 1) / 2), 2, 1};
    if (chunks <= 4 * R8_MAX_WARPS) return {(int)((chunks + 3) / 4), 4, 1};
    return {0, 0, 0};
}
static int r8_bytes(int dt) { return dt == MMB_F32 ? 4 : 2; }
static bool r8_type(int dt) { return dt == MMB_F32 || dt == MMB_BF16 || dt == MMB_F16; }
// 8 values of every row start on a 16-byte boundary
static bool r8_aligned(const void* p, int64_t stride, int bytes) {
    return !p || (((uintptr_t)p & 15) == 0 && (stride * bytes) % 16 == 0);
}
static bool r8_aligned_q(const void* p, int64_t stride) {
    return !p || (((uintptr_t)p & 7) == 0 && stride % 8 == 0);
}

template <class EX, class ER, bool VEC, bool CK>
static int r8_fwd_launch(const R8Fwd& p, const R8Shape& s, cudaStream_t st) {
    const dim3 block(32 * s.warps, s.half ? s.rows / 2 : s.rows);
    const unsigned grid = (unsigned)((p.rows + s.rows - 1) / s.rows);
    if constexpr (VEC)
        if (s.half) {
            r8_fwd_kernel<EX, ER, true, 1, 128, CK, 16><<<grid, block, 0, st>>>(p);
            return mmb_launch_status();
        }
    if (s.nc == 1) r8_fwd_kernel<EX, ER, VEC, 1, 128, CK><<<grid, block, 0, st>>>(p);
    else if (s.nc == 2 && s.warps == 1)
        r8_fwd_kernel<EX, ER, VEC, 2, 128, CK><<<grid, block, 0, st>>>(p);
    else if (s.nc == 2) r8_fwd_kernel<EX, ER, VEC, 2, 512, CK><<<grid, block, 0, st>>>(p);
    else if (s.warps > 1) r8_fwd_kernel<EX, ER, VEC, 4, 512, CK><<<grid, block, 0, st>>>(p);
    else if constexpr (VEC) r8_fwd_kernel<EX, ER, VEC, 4, 128, CK><<<grid, block, 0, st>>>(p);
    return mmb_launch_status();
}
template <class EX, class ER>
static int r8_fwd_form(const R8Fwd& p, const R8Shape& s, bool vec, bool ck, cudaStream_t st) {
    if (vec) return ck ? r8_fwd_launch<EX, ER, true, true>(p, s, st)
                       : r8_fwd_launch<EX, ER, true, false>(p, s, st);
    return ck ? r8_fwd_launch<EX, ER, false, true>(p, s, st)
              : r8_fwd_launch<EX, ER, false, false>(p, s, st);
}
static int r8_fwd(const R8Fwd& p, int xt, int rt, bool ck, cudaStream_t st) {
    const int xb = r8_bytes(xt), rb = r8_bytes(rt);
    const bool vec = p.cols % 8 == 0 && r8_aligned(p.x, p.xs, xb) && r8_aligned(p.res, p.rs, rb) &&
                     r8_aligned(p.h, p.hs, rb) && r8_aligned(p.n, p.ns, r8_bytes(p.nt)) &&
                     r8_aligned(p.w, 0, 4) && r8_aligned_q(p.q, p.qs);
    const R8Shape s = r8_shape(p.cols, vec);
    if (!s.nc) return MMB_ERR_UNSUPPORTED;
    if (xt == MMB_F32) return r8_fwd_form<T8F32, T8F32>(p, s, vec, ck, st);
    if (xt == MMB_BF16)
        return rt == MMB_F32 ? r8_fwd_form<T8BF16, T8F32>(p, s, vec, ck, st)
                             : r8_fwd_form<T8BF16, T8BF16>(p, s, vec, ck, st);
    return rt == MMB_F32 ? r8_fwd_form<T8F16, T8F32>(p, s, vec, ck, st)
                         : r8_fwd_form<T8F16, T8F16>(p, s, vec, ck, st);
}
static int r8_fwd_check(const R8Fwd& p, int xt, int rt) {
    if (p.rows < 0 || p.cols <= 0 || p.rows > INT32_MAX || p.cols > INT32_MAX)
        return MMB_ERR_SHAPE;
    if (!r8_type(xt) || (rt != xt && rt != MMB_F32)) return MMB_ERR_UNSUPPORTED;
    if (p.rows == 0) return MMB_OK;
    if (!p.x) return MMB_ERR_NULL;
    if (p.xs < p.cols || (p.res && p.rs < p.cols) || (p.h && p.hs < p.cols) ||
        (p.n && p.ns < p.cols) || (p.q && p.qs < p.cols))
        return MMB_ERR_SHAPE;
    return MMB_OK;
}

// The backward's shape: with an fp32 stream (whatever the gradient of the norm is in),
// three or four chunks take two warps a row (65536 x 1024 fp32: 175 -> 157 us; bf16
// gradients, where one warp spilled: 153 -> 134).
static R8Shape r8_bwd_shape(int64_t cols, bool vec, bool dx_f32) {
    const int64_t chunks = (cols + R8_CHUNK - 1) / R8_CHUNK;
    return r8_shape(cols, vec && !(dx_f32 && (chunks == 3 || chunks == 4)));
}
// Blocks of the backward: enough to fill the GPU, few enough that the lines of
// partial sums stay small.
static int r8_bwd_blocks(int64_t rows, const R8Shape& s, bool vec) {
    const int64_t need = (rows + s.rows - 1) / s.rows;
    // as many as are resident at once: one more an SM waits for the others to end
    // (65536 x 1024 bf16, four blocks where three fit: 133 us)
    const int64_t most = 148 * (s.rows > 1 ? (vec ? 4 : 3) : s.warps < 16 ? 16 / s.warps : 1);
    return (int)min64(need, most);
}
template <class EN, class EX, bool VEC>
static int r8_bwd_launch(const R8Bwd& p, const R8Shape& s, int blocks, cudaStream_t st) {
    const dim3 block(32 * s.warps, s.half ? s.rows / 2 : s.rows);
    const size_t sm = s.rows > 1 ? (size_t)block.y * p.cols * sizeof(float) : 0;  // <= 16 KB
    if constexpr (VEC)
        if (s.half) {
            r8_bwd_kernel<EN, EX, true, 1, 2, 128, 16><<<blocks, block, sm, st>>>(p);
            return mmb_launch_status();
        }
    if (s.nc == 1) r8_bwd_kernel<EN, EX, VEC, 1, 4, 128><<<blocks, block, sm, st>>>(p);
    else if (s.nc == 2 && s.warps == 1)
        r8_bwd_kernel<EN, EX, VEC, 2, 2, 128><<<blocks, block, sm, st>>>(p);
    else if (s.nc == 2) r8_bwd_kernel<EN, EX, VEC, 2, VEC ? 2 : 1, 512><<<blocks, block, sm, st>>>(p);
    else if (s.warps > 1) r8_bwd_kernel<EN, EX, VEC, 4, 1, 512><<<blocks, block, sm, st>>>(p);
    else if constexpr (VEC && sizeof(typename EX::T) == 2)
        r8_bwd_kernel<EN, EX, VEC, 4, 1, 128><<<blocks, block, sm, st>>>(p);
    return mmb_launch_status();
}

}  // namespace mmb

using namespace mmb;

extern "C" int mmb_norm_q8(int64_t rows, int64_t cols, int32_t x_type, const void* x, int64_t ldx,
                           int32_t res_type, const void* residual, int64_t ldr,
                           const float* weight, float eps, int32_t norm, void* h, int64_t ldh,
                           int8_t* q, int64_t ldq, float* scale, mmb_stream_t stream) {
    MMB_NVTX("mmb_norm_q8");
    R8Fwd p{};
    p.rows = rows; p.cols = cols; p.x = x; p.xs = ldx; p.res = residual; p.rs = ldr;
    p.w = weight; p.h = h; p.hs = ldh; p.q = q; p.qs = ldq; p.scale = scale; p.eps = eps;
    p.norm = norm ? 1 : 0;
    const int c = r8_fwd_check(p, x_type, res_type);
    if (c != MMB_OK || rows == 0) return c;
    if (!q || !scale) return MMB_ERR_NULL;
    return r8_fwd(p, x_type, res_type, false, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int mmb_norm_ck8_fwd(int64_t rows, int64_t cols, int32_t x_type, const void* x,
                                int64_t ldx, int32_t res_type, const void* residual, int64_t ldr,
                                const float* weight, float eps, int32_t norm, void* h, int64_t ldh,
                                int32_t n_type, void* n, int64_t ldn, int8_t* q, int64_t ldq, float* scale,
                                float* rstd, mmb_stream_t stream) {
    MMB_NVTX("mmb_norm_ck8_fwd");
    R8Fwd p{};
    p.rows = rows; p.cols = cols; p.x = x; p.xs = ldx; p.res = residual; p.rs = ldr;
    p.w = weight; p.h = h; p.hs = ldh; p.n = n; p.ns = ldn; p.nt = n_type; p.q = q; p.qs = ldq; p.scale = scale;
    p.rstd = rstd; p.eps = eps; p.norm = norm ? 1 : 0;
    const int c = r8_fwd_check(p, x_type, res_type);
    if (c != MMB_OK || rows == 0) return c;
    if ((q && !scale) || (!q && !n)) return MMB_ERR_NULL;
    if (n && !r8_type(n_type)) return MMB_ERR_UNSUPPORTED;
    return r8_fwd(p, x_type, res_type, true, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" size_t mmb_norm_ck8_bwd_work_floats(int64_t rows, int64_t cols) {
    if (rows <= 0 || cols <= 0) return 0;
    // the loads' form is not known here: the larger of the two (every shape of the
    // backward is one of r8_shape's)
    const R8Shape a = r8_shape(cols, false), b = r8_shape(cols, true);
    if (!a.nc) return 0;
    const int na = r8_bwd_blocks(rows, a, false), nb = r8_bwd_blocks(rows, b, true);
    return (size_t)(na > nb ? na : nb) * (size_t)cols;
}

extern "C" int mmb_norm_ck8_bwd(int64_t rows, int64_t cols, int32_t dn_type, const void* dn,
                                int64_t lddn, int32_t dx_type, const void* dh, int64_t lddh,
                                const float* weight, const int8_t* q, int64_t ldq,
                                const float* scale, const float* rstd, void* dx, int64_t lddx,
                                float* dweight, float* work, mmb_stream_t stream) {
    MMB_NVTX("mmb_norm_ck8_bwd");
    if (rows < 0 || cols <= 0 || rows > INT32_MAX || cols > INT32_MAX) return MMB_ERR_SHAPE;
    if (!r8_type(dn_type) || (dx_type != dn_type && dx_type != MMB_F32)) return MMB_ERR_UNSUPPORTED;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (rows == 0) {
        if (dweight && cudaMemsetAsync(dweight, 0, (size_t)cols * sizeof(float), st) != cudaSuccess)
            return mmb_launch_status();
        return MMB_OK;
    }
    if (!dn || !q || !scale || !rstd || !dx) return MMB_ERR_NULL;
    if (dweight && !work) return MMB_ERR_WORKSPACE;
    if (lddn < cols || (dh && lddh < cols) || ldq < cols || lddx < cols) return MMB_ERR_SHAPE;
    R8Bwd p{};
    p.rows = rows; p.cols = cols; p.dn = dn; p.dns = lddn; p.dh = dh; p.dhs = lddh; p.w = weight;
    p.q = q; p.qs = ldq; p.scale = scale; p.rstd = rstd; p.dx = dx; p.dxs = lddx;
    p.part = dweight ? work : nullptr;
    const int nb = r8_bytes(dn_type), xb = r8_bytes(dx_type);
    const bool vec = cols % 8 == 0 && r8_aligned(dn, lddn, nb) && r8_aligned(dh, lddh, xb) &&
                     r8_aligned(dx, lddx, xb) && r8_aligned(weight, 0, 4) && r8_aligned_q(q, ldq);
    const R8Shape s = r8_bwd_shape(cols, vec, dx_type == MMB_F32);
    if (!s.nc) return MMB_ERR_UNSUPPORTED;
    const int blocks = r8_bwd_blocks(rows, s, vec);
    int rc;
#define R8_BWD(EN, EX)                                                \
    (vec ? r8_bwd_launch<EN, EX, true>(p, s, blocks, st)              \
         : r8_bwd_launch<EN, EX, false>(p, s, blocks, st))
    if (dn_type == MMB_F32) rc = R8_BWD(T8F32, T8F32);
    else if (dn_type == MMB_BF16) rc = dx_type == MMB_F32 ? R8_BWD(T8BF16, T8F32) : R8_BWD(T8BF16, T8BF16);
    else rc = dx_type == MMB_F32 ? R8_BWD(T8F16, T8F32) : R8_BWD(T8F16, T8F16);
#undef R8_BWD
    if (rc != MMB_OK || !dweight) return rc;
    r8_colsum_kernel<<<(unsigned)((cols + R8_SUM_COLS - 1) / R8_SUM_COLS),
                       dim3(R8_SUM_COLS, R8_SUM_ROWS), 0, st>>>(
        work, blocks, cols, dweight);
    return mmb_launch_status();
}

extern "C" int mmb_restore_q8(int64_t rows, int64_t cols, const int8_t* q, int64_t ldq,
                              const float* scale, int32_t grouped, int32_t out_type, void* out,
                              int64_t ldo, mmb_stream_t stream) {
    MMB_NVTX("mmb_restore_q8");
    if (rows < 0 || cols <= 0 || rows > INT32_MAX || cols > INT32_MAX) return MMB_ERR_SHAPE;
    if (!r8_type(out_type)) return MMB_ERR_UNSUPPORTED;
    if (rows == 0) return MMB_OK;
    if (!q || !scale || !out) return MMB_ERR_NULL;
    if (ldq < cols || ldo < cols) return MMB_ERR_SHAPE;
    const int64_t chunks = (cols + R8_CHUNK - 1) / R8_CHUNK;
    if (chunks > 65535) return MMB_ERR_UNSUPPORTED;
    const dim3 blocks((unsigned)((rows + 8 * R8_RROWS - 1) / (8 * R8_RROWS)), (unsigned)chunks);
    const int64_t groups = grouped ? (cols + R8_GROUP - 1) / R8_GROUP : 0;
    const bool vec = cols % 8 == 0 && r8_aligned(out, ldo, r8_bytes(out_type)) && r8_aligned_q(q, ldq);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
#define R8_RESTORE(E)                                                                           \
    do {                                                                                        \
        if (vec)                                                                                \
            r8_restore_kernel<E, true><<<blocks, 256, 0, st>>>(rows, cols, q, ldq, scale,       \
                                                               groups, out, ldo);               \
        else                                                                                    \
            r8_restore_kernel<E, false><<<blocks, 256, 0, st>>>(rows, cols, q, ldq, scale,      \
                                                                groups, out, ldo);              \
    } while (0)
    if (out_type == MMB_F32) R8_RESTORE(T8F32);
    else if (out_type == MMB_BF16) R8_RESTORE(T8BF16);
    else R8_RESTORE(T8F16);
#undef R8_RESTORE
    return mmb_launch_status();
}
