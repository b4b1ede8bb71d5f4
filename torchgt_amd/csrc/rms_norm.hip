// Residual add and root-mean-square norm in one pass, its backward, and the norm (or any matrix) with an output in 8 bits.
//
//   s = x (+ r), rounded to the tensors' type;  y = s rstd w,  rstd = 1 / sqrt(mean(s^2) + eps)
//   ds = rstd (g - xhat mean(g xhat)) (+ extra),  g = dy w,  xhat = s rstd;   dw = sum over rows of dy xhat
//   8 bits: code = e4m3(y / scale), scale = the smallest power of two with max|y| <= 448 scale
//
// No counterpart in the reference (its layers have LayerNorm, models/graphormer_dist_node_level.py:280,284).  The norm is of s as it is stored: the backward
// reads that s.  Statistics and column sums are float32.  A power of two as a scale costs none of the codes' bits - they have an exponent of their
// own - and rounds nothing, where max|y| / 448 would round every value once more and put many on the borders between two codes.
//
// Bound by memory: every tensor is read and written once, in 16-byte pieces.  A row of up to 64 pieces is held by as many lanes as it has pieces (a power of
// two), a longer one by a wave with 2 or 4 pieces a lane, by a workgroup from 257 pieces on.
// Measured: 16384 x 2048 bf16 with a residual, forward 45.5 us and backward 45.4 us (268 MB each, 5.9 TB/s; a large copy reaches 5.0), sums over rows 4; 64000 x 64
// float32 12.5 and 13.6 (66 MB, 82 MB); 8191 x 1408 to 8 bits 16.7 (81 MB); one row of 1024 2.6.  Stores and loads past the caches (non-temporal) were slower.
#include "common.h"
#include <algorithm>

namespace tgt {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
struct b16 { uint16_t x; };

template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Loose { u32x4 v; };      // 16 bytes at any element's address

// One 16-byte piece of a row as floats
template <typename T> struct Vec;
template <> struct Vec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void unpack(u32x4 v, float (&f)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(v[i]);
    }
    static __device__ __forceinline__ u32x4 pack(const float (&f)[4]) {
        return u32x4{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
    }
    static __device__ __forceinline__ float rounded(float v) { return v; }
};
template <> struct Vec<b16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void unpack(u32x4 v, float (&f)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(v[i] << 16);
            f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ uint32_t bits(float v) { return __builtin_bit_cast(uint16_t, static_cast<__bf16>(v)); }
    static __device__ __forceinline__ u32x4 pack(const float (&f)[8]) {
        u32x4 o;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = bits(f[2 * i]) | bits(f[2 * i + 1]) << 16;
        return o;
    }
    static __device__ __forceinline__ float rounded(float v) { return __uint_as_float(bits(v) << 16); }
};

// Pieces of a row from element `at` on; zero from C on.  ALIGNED: C and every row's address are multiples of 16 bytes.
template <typename T, bool ALIGNED> __device__ __forceinline__ void load(const T* row, int at, int C, float (&f)[Vec<T>::N]) {
    constexpr int VE = Vec<T>::N;
    u32x4 v = {0u, 0u, 0u, 0u};
    if (ALIGNED) {
        if (at < C) v = *reinterpret_cast<const u32x4*>(row + at);
    } else if (at + VE <= C) {
        v = reinterpret_cast<const Loose<T>*>(row + at)->v;
    } else {
        union { T e[VE]; u32x4 v; } u;
        u.v = v;
        for (int i = 0; i < VE; ++i)
            if (at + i < C) u.e[i] = row[at + i];
        v = u.v;
    }
    Vec<T>::unpack(v, f);
}
template <typename T, bool ALIGNED> __device__ __forceinline__ void store(T* row, int at, int C, const float (&f)[Vec<T>::N]) {
    constexpr int VE = Vec<T>::N;
    const u32x4 v = Vec<T>::pack(f);
    if (ALIGNED) {
        if (at < C) *reinterpret_cast<u32x4*>(row + at) = v;
    } else if (at + VE <= C) {
        reinterpret_cast<Loose<T>*>(row + at)->v = v;
    } else {
        union { T e[VE]; u32x4 v; } u;
        u.v = v;
        for (int i = 0; i < VE; ++i)
            if (at + i < C) row[at + i] = u.e[i];
    }
}

// Sum / largest value over the LPR threads of a row, for all of them.  More than a wave: through LDS (every thread of the workgroup calls it).
template <int LPR, bool MAX> __device__ __forceinline__ float over_row(float v, float* red) {
#pragma unroll
    for (int o = (LPR < 64 ? LPR : 64) / 2; o > 0; o >>= 1) {
        const float t = __shfl_xor(v, o, 64);
        v = MAX ? fmaxf(v, t) : v + t;
    }
    if constexpr (LPR > 64) {
        __syncthreads();      // (the values of the call before have been read)
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int w = 1; w < LPR / 64; ++w) v = MAX ? fmaxf(v, red[w]) : v + red[w];
    }
    return v;
}

// LPR threads and NV pieces each to a row, BT threads to a workgroup
template <int LPR_, int NV_> struct Rows {
    static constexpr int LPR = LPR_, NV = NV_, BT = LPR_ > 256 ? LPR_ : 256, RPB = BT / LPR_;
};

// s and y, or (EIGHT) s and codes with scales; NORM false: codes of x itself
template <typename T, typename R, bool ALIGNED, bool EIGHT, bool NORM>
__global__ __launch_bounds__(R::BT) void k_rms_fwd(const T* __restrict__ x, const T* __restrict__ r, const T* __restrict__ weight, int64_t N, int C, float eps,
                                                   T* __restrict__ sum_out, T* __restrict__ y, float* __restrict__ rstd_out, uint8_t* __restrict__ codes,
                                                   float* __restrict__ scales) {
    constexpr int VE = Vec<T>::N, LPR = R::LPR, NV = R::NV;
    __shared__ float red[R::BT / 64];
    const int sub = threadIdx.x % LPR, slot = threadIdx.x / LPR;
    for (int64_t row = (int64_t)blockIdx.x * R::RPB + slot; row < N; row += (int64_t)gridDim.x * R::RPB) {
        float s[NV][VE], w[NV][VE];
#pragma unroll
        for (int i = 0; i < NV; ++i) load<T, ALIGNED>(x + row * C, (sub + i * LPR) * VE, C, s[i]);
        if (NORM) {
#pragma unroll
            for (int i = 0; i < NV; ++i) load<T, ALIGNED>(weight, (sub + i * LPR) * VE, C, w[i]);
        }
        if (r) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                float t[VE];
                load<T, ALIGNED>(r + row * C, (sub + i * LPR) * VE, C, t);
#pragma unroll
                for (int e = 0; e < VE; ++e) s[i][e] = Vec<T>::rounded(s[i][e] + t[e]);
                store<T, ALIGNED>(sum_out + row * C, (sub + i * LPR) * VE, C, s[i]);
            }
        }
        if (NORM) {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < VE; ++e) ss += s[i][e] * s[i][e];
            const float rstd = 1.f / sqrtf(over_row<LPR, false>(ss, red) / (float)C + eps);      // (rsqrtf is off by up to an ulp, for a whole row)
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < VE; ++e) s[i][e] = s[i][e] * rstd * w[i][e];
            if (rstd_out && sub == 0) rstd_out[row] = rstd;
        }
        if (!EIGHT) {
#pragma unroll
            for (int i = 0; i < NV; ++i) store<T, ALIGNED>(y + row * C, (sub + i * LPR) * VE, C, s[i]);
        } else {
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < VE; ++e) top = fmaxf(top, fabsf(s[i][e]));
            const uint32_t bits = __float_as_uint(over_row<LPR, true>(top, red));
            // 2^(e - 8) for up to 1.75 2^e (448 is 1.75 2^8), 2^(e - 7) above; no less than 2^-126, so that its inverse is a number too
            int k = (int)(bits >> 23) - 127 - ((bits & 0x7fffffu) > 0x600000u ? 7 : 8);
            k = k < -126 ? -126 : k;
            k = bits ? k : 0;
            const float inv = __uint_as_float((uint32_t)(127 - k) << 23);
            if (sub == 0) scales[row] = __uint_as_float((uint32_t)(127 + k) << 23);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                uint32_t c[VE / 4];
#pragma unroll
                for (int q = 0; q < VE / 4; ++q) {
                    int v = __builtin_amdgcn_cvt_pk_fp8_f32(s[i][4 * q] * inv, s[i][4 * q + 1] * inv, 0, false);
                    c[q] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(s[i][4 * q + 2] * inv, s[i][4 * q + 3] * inv, v, true);
                }
                const int at = (sub + i * LPR) * VE;
                uint8_t* to = codes + row * C + at;
                if (ALIGNED) {
                    if (at < C) {
                        if constexpr (VE == 8) *reinterpret_cast<uint2*>(to) = make_uint2(c[0], c[1]);
                        else *reinterpret_cast<uint32_t*>(to) = c[0];
                    }
                } else {
                    for (int e = 0; e < VE; ++e)
                        if (at + e < C) to[e] = (uint8_t)(c[e >> 2] >> (8 * (e & 3)));
                }
            }
        }
    }
}

// ds, and per-workgroup sums of dy xhat over its rows -> partial[blockIdx.x][C]
template <typename T, typename R, bool ALIGNED>
__global__ __launch_bounds__(R::BT) void k_rms_bwd(const T* __restrict__ s_in, const T* __restrict__ weight, const float* __restrict__ rstd_in,
                                                   const T* __restrict__ dy, const T* __restrict__ extra, int64_t N, int C, T* __restrict__ ds,
                                                   float* __restrict__ partial) {
    constexpr int VE = Vec<T>::N, LPR = R::LPR, NV = R::NV;
    __shared__ float red[R::BT / 64];
    __shared__ float cols[LPR > 64 ? 1 : (R::BT / 64) * (LPR < 64 ? LPR : 64) * NV * VE];
    const int sub = threadIdx.x % LPR, slot = threadIdx.x / LPR;
    float w[NV][VE], dw[NV][VE];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        load<T, ALIGNED>(weight, (sub + i * LPR) * VE, C, w[i]);
#pragma unroll
        for (int e = 0; e < VE; ++e) dw[i][e] = 0.f;
    }
    for (int64_t row = (int64_t)blockIdx.x * R::RPB + slot; row < N; row += (int64_t)gridDim.x * R::RPB) {
        float s[NV][VE], d[NV][VE], t[NV][VE];
#pragma unroll
        for (int i = 0; i < NV; ++i) load<T, ALIGNED>(s_in + row * C, (sub + i * LPR) * VE, C, s[i]);
#pragma unroll
        for (int i = 0; i < NV; ++i) load<T, ALIGNED>(dy + row * C, (sub + i * LPR) * VE, C, d[i]);
        if (extra) {
#pragma unroll
            for (int i = 0; i < NV; ++i) load<T, ALIGNED>(extra + row * C, (sub + i * LPR) * VE, C, t[i]);
        }
        const float rstd = rstd_in[row];
        float a = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const float xh = s[i][e] * rstd;
                dw[i][e] += d[i][e] * xh;
                s[i][e] = xh;
                d[i][e] *= w[i][e];
                a += d[i][e] * xh;
            }
        const float m = over_row<LPR, false>(a, red) / (float)C;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float o[VE];
#pragma unroll
            for (int e = 0; e < VE; ++e) o[e] = rstd * (d[i][e] - s[i][e] * m) + (extra ? t[i][e] : 0.f);
            store<T, ALIGNED>(ds + row * C, (sub + i * LPR) * VE, C, o);
        }
    }
    float* out = partial + (int64_t)blockIdx.x * C;
    if constexpr (LPR > 64) {      // one row at a time: a thread's sums are the workgroup's
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VE; ++e)
                if ((sub + i * LPR) * VE + e < C) out[(sub + i * LPR) * VE + e] = dw[i][e];
    } else {
        constexpr int kCols = LPR * NV * VE;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                float v = dw[i][e];
#pragma unroll
                for (int o = LPR; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);      // (the rows that the wave has side by side)
                if ((threadIdx.x & 63) < LPR) cols[(threadIdx.x >> 6) * kCols + (sub + i * LPR) * VE + e] = v;
            }
        __syncthreads();
        for (int c = threadIdx.x; c < C; c += R::BT) {
            float v = cols[c];
#pragma unroll
            for (int k = 1; k < R::BT / 64; ++k) v += cols[k * kCols + c];
            out[c] = v;
        }
    }
}

template <typename T> __global__ __launch_bounds__(256) void k_zero_row(T* __restrict__ p, int n) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < n) p[i] = T{};
}

constexpr int kMostFeatures = 16384;
constexpr int kBwdWorkers = 512;      // most workgroups (= partial sums) of the backward

int check_norm(int64_t N, int C, int dtype, const char* who) {
    if (N < 0 || C < 1 || (dtype != TGT_DTYPE_F32 && dtype != TGT_DTYPE_BF16)) {
        set_error("%s: bad size or dtype", who);
        return TGT_ERR_INVALID_ARG;
    }
    if (C > kMostFeatures) {
        set_error("%s: %d features, at most %d", who, C, kMostFeatures);
        return TGT_ERR_UNSUPPORTED;
    }
    return TGT_OK;
}

// X(Rows type) for rows of C elements of T
#define TGT_ROWS(T, C, X)                                                  \
    do {                                                                   \
        const int v_ = ((C) + Vec<T>::N - 1) / Vec<T>::N;                  \
        if (v_ <= 8) { using R = Rows<8, 1>; X }                           \
        else if (v_ <= 16) { using R = Rows<16, 1>; X }                    \
        else if (v_ <= 32) { using R = Rows<32, 1>; X }                    \
        else if (v_ <= 64) { using R = Rows<64, 1>; X }                    \
        else if (v_ <= 128) { using R = Rows<64, 2>; X }                   \
        else if (v_ <= 256) { using R = Rows<64, 4>; X }                   \
        else if (v_ <= 512) { using R = Rows<256, 2>; X }                  \
        else if (v_ <= 1024) { using R = Rows<256, 4>; X }                 \
        else if (v_ <= 2048) { using R = Rows<256, 8>; X }                 \
        else { using R = Rows<sizeof(T) == 4 ? 1024 : 256, sizeof(T) == 4 ? 4 : 8>; X } \
    } while (0)

unsigned blocks_for(int64_t N, int rpb, int most) { return (unsigned)std::max<int64_t>(1, std::min<int64_t>((N + rpb - 1) / rpb, most)); }
bool all16(std::initializer_list<const void*> ps) {
    for (const void* p : ps)
        if ((uintptr_t)p & 15) return false;
    return true;
}

template <typename T, bool EIGHT, bool NORM>
int launch_fwd(const void* x, const void* r, const void* w, int64_t N, int C, float eps, void* sum, void* y, float* rstd, void* codes, float* scales, hipStream_t st) {
    const bool al = C % Vec<T>::N == 0 && all16({x, r, w, sum, y, codes});
#define X                                                                                                                                            \
    {                                                                                                                                                \
        const dim3 grid(blocks_for(N, R::RPB, 8192));                                                                                                \
        if (al)                                                                                                                                      \
            hipLaunchKernelGGL((k_rms_fwd<T, R, true, EIGHT, NORM>), grid, dim3(R::BT), 0, st, (const T*)x, (const T*)r, (const T*)w, N, C, eps, (T*)sum, \
                               (T*)y, rstd, (uint8_t*)codes, scales);                                                                                \
        else                                                                                                                                         \
            hipLaunchKernelGGL((k_rms_fwd<T, R, false, EIGHT, NORM>), grid, dim3(R::BT), 0, st, (const T*)x, (const T*)r, (const T*)w, N, C, eps, (T*)sum, \
                               (T*)y, rstd, (uint8_t*)codes, scales);                                                                                \
    }
    TGT_ROWS(T, C, X);
#undef X
    TGT_HIP_CHECK(hipGetLastError());
    return TGT_OK;
}

template <typename T>
int launch_bwd(const void* s, const void* w, const float* rstd, const void* dy, const void* extra, int64_t N, int C, void* ds, float* partial, int* workers,
               hipStream_t st) {
    const bool al = C % Vec<T>::N == 0 && all16({s, w, dy, extra, ds});
#define X                                                                                                                                            \
    {                                                                                                                                                \
        const unsigned grid = blocks_for(N, R::RPB, kBwdWorkers);                                                                                    \
        *workers = (int)grid;                                                                                                                        \
        if (al)                                                                                                                                      \
            hipLaunchKernelGGL((k_rms_bwd<T, R, true>), dim3(grid), dim3(R::BT), 0, st, (const T*)s, (const T*)w, rstd, (const T*)dy, (const T*)extra, N, C, \
                               (T*)ds, partial);                                                                                                     \
        else                                                                                                                                         \
            hipLaunchKernelGGL((k_rms_bwd<T, R, false>), dim3(grid), dim3(R::BT), 0, st, (const T*)s, (const T*)w, rstd, (const T*)dy, (const T*)extra, N, C, \
                               (T*)ds, partial);                                                                                                     \
    }
    TGT_ROWS(T, C, X);
#undef X
    TGT_HIP_CHECK(hipGetLastError());
    return TGT_OK;
}

}  // namespace
}  // namespace tgt

extern "C" {

int tgt_add_rms_norm_fwd(const void* d_x, const void* d_r, const void* d_weight, int64_t N, int C, float eps, int dtype, void* d_sum, void* d_y, float* d_rstd,
                         void* stream) {
    using namespace tgt;
    const int rc = check_norm(N, C, dtype, "tgt_add_rms_norm_fwd");
    if (rc != TGT_OK || N == 0) return rc;
    if (!d_x || !d_weight || !d_y || (d_r && !d_sum)) { set_error("tgt_add_rms_norm_fwd: null pointer"); return TGT_ERR_INVALID_ARG; }
    hipStream_t st = (hipStream_t)stream;
    KernelTimer t(KS_LAYER_NORM_FWD, st);
    return dtype == TGT_DTYPE_F32 ? launch_fwd<float, false, true>(d_x, d_r, d_weight, N, C, eps, d_sum, d_y, d_rstd, nullptr, nullptr, st)
                                  : launch_fwd<b16, false, true>(d_x, d_r, d_weight, N, C, eps, d_sum, d_y, d_rstd, nullptr, nullptr, st);
}

int tgt_add_rms_norm_8bit(const void* d_x, const void* d_r, const void* d_weight, int64_t N, int C, float eps, int dtype, void* d_sum, void* d_codes,
                          float* d_scales, void* stream) {
    using namespace tgt;
    const int rc = check_norm(N, C, dtype, "tgt_add_rms_norm_8bit");
    if (rc != TGT_OK || N == 0) return rc;
    if (!d_x || !d_weight || !d_codes || !d_scales || (d_r && !d_sum)) { set_error("tgt_add_rms_norm_8bit: null pointer"); return TGT_ERR_INVALID_ARG; }
    hipStream_t st = (hipStream_t)stream;
    KernelTimer t(KS_LAYER_NORM_FWD, st);
    return dtype == TGT_DTYPE_F32 ? launch_fwd<float, true, true>(d_x, d_r, d_weight, N, C, eps, d_sum, nullptr, nullptr, d_codes, d_scales, st)
                                  : launch_fwd<b16, true, true>(d_x, d_r, d_weight, N, C, eps, d_sum, nullptr, nullptr, d_codes, d_scales, st);
}

int tgt_quantize_rows(const void* d_w, int64_t N, int C, int dtype, void* d_codes, float* d_scales, void* stream) {
    using namespace tgt;
    const int rc = check_norm(N, C, dtype, "tgt_quantize_rows");
    if (rc != TGT_OK || N == 0) return rc;
    if (!d_w || !d_codes || !d_scales) { set_error("tgt_quantize_rows: null pointer"); return TGT_ERR_INVALID_ARG; }
    hipStream_t st = (hipStream_t)stream;
    return dtype == TGT_DTYPE_F32 ? launch_fwd<float, true, false>(d_w, nullptr, nullptr, N, C, 0.f, nullptr, nullptr, nullptr, d_codes, d_scales, st)
                                  : launch_fwd<b16, true, false>(d_w, nullptr, nullptr, N, C, 0.f, nullptr, nullptr, nullptr, d_codes, d_scales, st);
}

int64_t tgt_rms_norm_bwd_workspace_bytes(int64_t N, int C) {
    if (N < 0 || C < 1) return -1;
    return (int64_t)sizeof(float) * C * std::min<int64_t>(N, tgt::kBwdWorkers);
}

int tgt_rms_norm_bwd(const void* d_s, const void* d_weight, const float* d_rstd, const void* d_dy, const void* d_ds_extra, int64_t N, int C, int dtype, void* d_ds,
                     void* d_dweight, void* d_workspace, int64_t workspace_bytes, void* stream) {
    using namespace tgt;
    const int rc = check_norm(N, C, dtype, "tgt_rms_norm_bwd");
    if (rc != TGT_OK) return rc;
    hipStream_t st = (hipStream_t)stream;
    if (!d_dweight) { set_error("tgt_rms_norm_bwd: null pointer"); return TGT_ERR_INVALID_ARG; }
    if (N == 0) {
        const dim3 grid((unsigned)((C + 255) / 256));
        if (dtype == TGT_DTYPE_F32) hipLaunchKernelGGL((k_zero_row<float>), grid, dim3(256), 0, st, (float*)d_dweight, C);
        else hipLaunchKernelGGL((k_zero_row<b16>), grid, dim3(256), 0, st, (b16*)d_dweight, C);
        TGT_HIP_CHECK(hipGetLastError());
        return TGT_OK;
    }
    if (!d_s || !d_weight || !d_rstd || !d_dy || !d_ds) { set_error("tgt_rms_norm_bwd: null pointer"); return TGT_ERR_INVALID_ARG; }
    if (!d_workspace || workspace_bytes < tgt_rms_norm_bwd_workspace_bytes(N, C) || ((uintptr_t)d_workspace & 15)) {
        set_error("tgt_rms_norm_bwd: workspace of %lld bytes (16-byte aligned) needed, got %lld", (long long)tgt_rms_norm_bwd_workspace_bytes(N, C),
                  (long long)workspace_bytes);
        return TGT_ERR_WORKSPACE;
    }
    int workers = 0;
    {
        KernelTimer t(KS_LAYER_NORM_BWD, st);
        const int err = dtype == TGT_DTYPE_F32 ? launch_bwd<float>(d_s, d_weight, d_rstd, d_dy, d_ds_extra, N, C, d_ds, (float*)d_workspace, &workers, st)
                                               : launch_bwd<b16>(d_s, d_weight, d_rstd, d_dy, d_ds_extra, N, C, d_ds, (float*)d_workspace, &workers, st);
        if (err != TGT_OK) return err;
    }
    tgt_reduce_desc r{};
    r.partial = (float*)d_workspace; r.workers = workers; r.n = C; r.n_out = 1;
    r.out[0] = d_dweight;
    return reduce_partials(&r, 1, dtype, st);
}

}  // extern "C"
