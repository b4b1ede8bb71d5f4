// The gated projections of a feed-forward block and linears with an epilogue, forward and backward, for matrices of any size:
//
//   gated   h = act(x Wg^T + bg) * (x Wu^T + bu)          both products, the activation and the product of the two in one kernel
//   linear  y = act(x W^T + b) + residual
//
// No counterpart in the reference, whose feed-forward block has one projection and a GELU (models/graphormer_dist_node_level.py:27-39).
//
// Backward.  With g = x Wg^T + bg, u = x Wu^T + bu:  dg = dh u act'(g), du = dh act(g);  dx = dg Wg + du Wu;  dWg = dg^T x, dWu = du^T x; biases: column
// sums.  Where the contraction is long the forward keeps g and u (bfloat16: 14 bits and an exponent for four; h is formed of the
// float32 values); where it is short they are not kept: a first kernel forms them again in float32.  Either writes dg and du, rounded to the tensors' type since
// they are operands of the next two products; dx and dW are products of what it wrote.  A product of few output tiles is cut along its contraction, partial sums in float32 added in a fixed order.
//
// Measured (us; 2 n N K F operations and what a large library product of the same type reaches, 1422 TFLOP/s in bf16): gated 16384 x 1024 x 4096 bf16 forward
// with kept values 300 to 333 (193; without kept values 266), kept gradients 149 (671 MB at 4.5 TB/s), input gradient 205 to 226 (193), weight gradients 238 to 262 (193):
// a hot card is slower.  linear 16384 x 4096 x 1024: 114 to 129, 129 to 139, 136 to 146 (97 each).  8 bits, 4099 x 1024 x 2816 gated: 35 (18).
#include "activations.h"
#include "block_gemm.h"
#include "gated_tiles.h"
#include <algorithm>

namespace tgt {
namespace {

using namespace gemm;

// Four neighbouring elements of a row in memory
template <typename O> struct Four { O e[4]; };
template <> struct Four<b16> { union { b16 e[4]; uint2 v; }; };
template <> struct Four<float> { union { float e[4]; u32x4 v; }; };
// WHOLE: all four exist and the address is aligned to them; else the first n do
template <typename O, bool WHOLE> __device__ __forceinline__ Four<O> load4(const O* p, int n) {
    Four<O> f;
    if constexpr (WHOLE) f.v = *reinterpret_cast<const decltype(f.v)*>(p);
    else {
        f.v = decltype(f.v){};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < n) f.e[i] = p[i];
    }
    return f;
}
template <typename O, bool WHOLE> __device__ __forceinline__ void store4(O* p, int n, const float (&v)[4]) {
    Four<O> f;
#pragma unroll
    for (int i = 0; i < 4; ++i) from_float(f.e[i], v[i]);
    if constexpr (WHOLE) *reinterpret_cast<decltype(f.v)*>(p) = f.v;
    else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < n) p[i] = f.e[i];
    }
}
template <typename O> __device__ __forceinline__ bool sixteens(const void* p, int64_t ld) { return ((uintptr_t)p & 15) == 0 && ld * sizeof(O) % 16 == 0; }

// Four columns of two neighbouring pieces of 16 become eight columns of one: lanes of the first and third 16 then have the first piece, the others the second
// (and back: the exchange is its own inverse)
__device__ __forceinline__ void exchange(uint2& first, uint2& second) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    const u32x2 x = __builtin_amdgcn_permlane16_swap(first.x, second.x, false, false), y = __builtin_amdgcn_permlane16_swap(first.y, second.y, false, false);
    first = make_uint2(x[0], y[0]);
    second = make_uint2(x[1], y[1]);
}

// Four neighbouring values for the backward in the room of four bf16: one exponent, that of the largest, and 14 bits each, off by at most 2^-13 of the
// largest.  What the gradients are formed of would otherwise be rounded as coarsely as they are themselves (bf16, 16384 x 1024 x 4096: the gradients off by 0.0030 instead of
// 0.0023; 0.0017 is their own last rounding).  Values below 2^-114 lose bits; beside an infinity or a NaN each has sign, exponent and 5 bits of its own.
// SIGNS: none but zeros become zero (an activation with an edge there), off by less than a step then, 2^-12 of the largest.
template <bool SIGNS> __device__ __forceinline__ uint2 pack_four(const float (&v)[4]) {
    uint32_t b[4], m[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(v[i]);
    const uint32_t top = max(max(b[0] & 0x7fffffffu, b[1] & 0x7fffffffu), max(b[2] & 0x7fffffffu, b[3] & 0x7fffffffu)), exponent = max(top >> 23, 13u);
    const float scale = __uint_as_float((266 - exponent) << 23), at = 12582912.f;      // (1.5 2^23: the sum's low bits are the rounded product)
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = __float_as_uint(__builtin_amdgcn_fmed3f(__builtin_fmaf(v[i], scale, at), at - 8191.f, at + 8191.f));
    if constexpr (SIGNS) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (m[i] == __float_as_uint(at) && v[i] != 0.f) m[i] += v[i] < 0.f ? -1 : 1;
    }
    if (__builtin_expect(exponent == 255, 0)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) m[i] = (v[i] != v[i] ? b[i] | 0x400000u : b[i]) >> 18;
    }
    const auto select = [](uint32_t mask, uint32_t x, uint32_t y) { return (x & mask) | (y & ~mask); };      // one instruction
    return make_uint2(select(0x3fffu, m[0], select(0xfffffffu, m[1] << 14, m[2] << 28)), select(0x3ffu, m[2] >> 4, select(0xffffffu, m[3] << 10, exponent << 24)));
}
__device__ __forceinline__ void unpack_four(uint2 p, float (&v)[4]) {
    const uint32_t exponent = p.y >> 24, m[4] = {p.x << 18, p.x >> 14 << 18, p.x >> 28 << 18 | p.y << 22, p.y >> 10 << 18};      // from the highest bit on
    if (__builtin_expect(exponent == 255, 0)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(m[i]);
    } else {
        const float scale = __uint_as_float((exponent - 12) << 23);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (float)((int)m[i] >> 18) * scale;
    }
}
// elements of a row of one weight's kept values
template <typename O> __host__ __device__ __forceinline__ int64_t kept_width(int64_t F) { return sizeof(O) == 2 ? (F + 3) / 4 * 4 : F; }

// What becomes of a tile's sums.  WHOLE: the tile lies inside the result and all rows are aligned to 16 bytes; what is read is then asked for before the
// first value is formed, and 16-bit rows are read and written 16 bytes a lane, 64 in a row, by an exchange between the pieces (8 bytes a lane: 16 rows of 32 bytes an
// instruction).
template <typename T, typename O, int FORM, bool TWO, bool GRAD, typename S, int ACT, bool WHOLE>
__device__ __forceinline__ void finish(const Args& a, int64_t p0, int64_t q0, unsigned split, const f32x4 (&acc)[S::FP][S::FQ]) {
    constexpr bool kPair = FORM == kForward && TWO, EXACT = sizeof(O) == 4, kReads = FORM == kForward && (GRAD || !TWO);
    constexpr int kBy = kPair ? 2 : 1, kOut = S::FP / kBy;      // pieces that one output piece takes
    constexpr bool kWide = WHOLE && sizeof(O) == 2 && kOut % 2 == 0;
    constexpr bool kKeeps = FORM == kForward && !GRAD && sizeof(T) > 1;
    constexpr int kGroup = kWide ? 2 : 1;
    const int lane = fresh_lane(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = (lane >> 4) * 4, row = lane & 15;
    const int wide_col = ((lane >> 4) & 1) * 16 + (lane >> 5) * 8;      // of 32
    const O* more = reinterpret_cast<const O*>(GRAD ? a.dy : a.residual);
    const bool to_partial = FORM == kWeightGrad && a.partial;
    int left[kOut];
#pragma unroll
    for (int i = 0; i < kOut; ++i) {
        const int64_t n = a.p_count - (p0 + S::p_piece(wave, i * kBy) / kBy * 16 + col);
        left[i] = n < 4 ? (int)n : 4;
        if (S::kUsed < 16 && col >= S::kUsed) left[i] = 0;
    }
    Four<O> in[kReads ? kOut : 1][S::FQ];
    if (kReads && more) {
#pragma unroll
        for (int j = 0; j < S::FQ; ++j) {
            const int64_t q = q0 + S::q_piece(wave, j) * 16 + row;
            const O* from = more + q * a.p_count + p0;
#pragma unroll
            for (int i = 0; i < kOut; i += kGroup) {
                const O* at = from + S::p_piece(wave, i * kBy) / kBy * 16;
                if constexpr (kWide && kReads) {
                    const u32x4 v = *reinterpret_cast<const u32x4*>(at + wide_col);
                    in[i][j].v = make_uint2(v.x, v.y);
                    in[i + 1][j].v = make_uint2(v.z, v.w);
                } else in[kReads ? i : 0][j] = load4<O, WHOLE>(at + col, q < a.q_count ? left[i] : 0);
            }
        }
    }
#pragma unroll
    for (int i0 = 0; i0 < kOut; i0 += kGroup) {
        float bias[kGroup][kBy][4], scale[kGroup][kBy][4];
        if constexpr (FORM == kForward) {
#pragma unroll
            for (int n = 0; n < kGroup; ++n) {
                const int64_t p = p0 + S::p_piece(wave, (i0 + n) * kBy) / kBy * 16 + col;
#pragma unroll
                for (int w = 0; w < kBy; ++w) {
                    Four<O> b;
                    Four<float> s;
                    b.v = decltype(b.v){};
                    if (a.bias[w]) b = load4<O, false>(reinterpret_cast<const O*>(a.bias[w]) + p, left[i0 + n]);
                    if constexpr (sizeof(T) == 1) s = load4<float, false>(a.p_scale[w] + p, left[i0 + n]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        bias[n][w][e] = to_float(b.e[e]);
                        if constexpr (sizeof(T) == 1) scale[n][w][e] = s.e[e];
                    }
                }
            }
        }
#pragma unroll
        for (int j = 0; j < S::FQ; ++j) {
            const int64_t q = q0 + S::q_piece(wave, j) * 16 + row;
            if (!WHOLE && (q >= a.q_count || row >= S::kUsed)) continue;
            if constexpr (kWide && kReads) {
                if (more) exchange(in[i0][j].v, in[i0 + 1][j].v);
            }
            float o[kGroup][4], o2[kGroup][4], keep[kBy][kGroup][4];
#pragma unroll
            for (int n = 0; n < kGroup; ++n) {
                const int i = i0 + n;
                if constexpr (FORM == kForward) {
                    float v[kBy][4];
                    const float qs = sizeof(T) == 1 ? a.q_scale[q] : 1.f;
#pragma unroll
                    for (int w = 0; w < kBy; ++w)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float t = acc[i * kBy + w][j][e];
                            if constexpr (sizeof(T) == 1) t *= qs * scale[n][w][e];
                            v[w][e] = t + bias[n][w][e];
                            if constexpr (kKeeps) keep[w][n][e] = v[w][e];
                        }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if constexpr (GRAD && kPair) {
                            const float dy = to_float(in[i][j].e[e]);
                            float f, s;
                            act_and_slope<EXACT, ACT>(v[0][e], f, s);
                            o[n][e] = dy * v[kBy - 1][e] * s;
                            o2[n][e] = dy * f;
                        } else if constexpr (GRAD) {
                            o[n][e] = slope_of<EXACT, ACT>(v[0][e], to_float(in[i][j].e[e]));
                        } else {
                            o[n][e] = act_of<EXACT, ACT>(v[0][e]);
                            if constexpr (kPair) o[n][e] *= v[1][e];
                            else if (more) o[n][e] += to_float(in[i][j].e[e]);
                        }
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[n][e] = acc[i][j][e];
                }
            }
            const int64_t p = p0 + S::p_piece(wave, i0 * kBy) / kBy * 16;
            const auto put = [&](O* out, const float (&v)[kGroup][4]) {
                if constexpr (kWide) {
                    Four<O> f[2];
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) from_float(f[n].e[e], v[kGroup - 2 + n][e]);
                    exchange(f[0].v, f[1].v);
                    *reinterpret_cast<u32x4*>(out + wide_col) = u32x4{f[0].v.x, f[0].v.y, f[1].v.x, f[1].v.y};
                } else store4<O, WHOLE>(out + col, left[i0], v[0]);
            };
            if (to_partial) {
                float* out = a.partial + ((int64_t)split * a.q_count + q) * a.p_count + p + col;
#pragma unroll
                for (int n = 0; n < kGroup; ++n) store4<float, WHOLE>(out + 16 * n, left[i0 + n], o[n]);
            } else if (FORM == kWeightGrad && q >= a.q_first) {
                put(reinterpret_cast<O*>(a.out[1]) + (q - a.q_first) * a.out_ld + p, o);
            } else {
                put(reinterpret_cast<O*>(a.out[0]) + q * a.out_ld + p, o);
                if constexpr (kKeeps) {
                    if (a.kept) {
                        const int64_t width = kept_width<O>(a.p_count);
                        O* to = reinterpret_cast<O*>(a.kept) + q * (kBy * width) + p;
#pragma unroll
                        for (int w = 0; w < kBy; ++w, to += width) {
                            if constexpr (sizeof(O) == 2) {
                                uint2 f[kGroup];
#pragma unroll
                                for (int n = 0; n < kGroup; ++n) {
                                    if constexpr (!WHOLE) {
#pragma unroll
                                        for (int e = 0; e < 4; ++e)
                                            if (e >= left[i0 + n]) keep[w][n][e] = 0.f;
                                    }
                                    f[n] = pack_four<ACT == TGT_ACT_RELU>(keep[w][n]);
                                }
                                if constexpr (kWide) {
                                    exchange(f[0], f[kGroup - 1]);
                                    *reinterpret_cast<u32x4*>(to + wide_col) = u32x4{f[0].x, f[0].y, f[kGroup - 1].x, f[kGroup - 1].y};
                                } else if (WHOLE || left[i0] > 0) *reinterpret_cast<uint2*>(to + col) = f[0];
                            } else put(to, keep[w]);
                        }
                    }
                }
                if constexpr (GRAD && kPair) put(reinterpret_cast<O*>(a.out[1]) + q * a.out_ld + p, o2);
            }
        }
    }
}
template <typename T, typename O, int FORM, bool TWO, bool GRAD, typename S>
__device__ __forceinline__ void epilogue(const Args& a, int64_t p0, int64_t q0, unsigned split, const f32x4 (&acc)[S::FP][S::FQ]) {
    constexpr int kCols = FORM == kForward && TWO ? S::kCols / 2 : S::kCols;
    const void* more = GRAD ? a.dy : a.residual;
    const bool whole = S::kUsed == 16 && p0 + kCols <= a.p_count && q0 + S::kRows <= a.q_count &&
                       (FORM == kWeightGrad && a.partial ? sixteens<float>(a.partial, a.p_count) : sixteens<O>(a.out[0], a.out_ld) && sixteens<O>(a.out[1], a.out_ld)) &&
                       (!more || sixteens<O>(more, a.p_count)) && sixteens<O>(a.kept, a.p_count);
#define X(ACT) do { if (whole) finish<T, O, FORM, TWO, GRAD, S, ACT, true>(a, p0, q0, split, acc); else finish<T, O, FORM, TWO, GRAD, S, ACT, false>(a, p0, q0, split, acc); } while (0)
    if constexpr (FORM != kForward) {
        X(TGT_ACT_NONE);
    } else {
        switch (a.act) {
            case TGT_ACT_SILU: X(TGT_ACT_SILU); break;
            case TGT_ACT_GELU: X(TGT_ACT_GELU); break;
            case TGT_ACT_RELU: X(TGT_ACT_RELU); break;
            default: X(TGT_ACT_NONE); break;
        }
    }
#undef X
}

template <typename T, typename O, int FORM, bool TWO, bool GRAD, bool ALIGNED, typename S, int STAGES>
__global__ __launch_bounds__(S::kThreads) void k_product(const Args a, const unsigned splits) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    unsigned tp, tq, split;
    if (!tile_of(a, splits, blockIdx.x, tp, tq, split)) return;
    const int64_t p0 = (int64_t)tp * (FORM == kForward && TWO ? S::kCols / 2 : S::kCols), q0 = (int64_t)tq * S::kRows;
    const int64_t k0 = (int64_t)split * a.K_each, k1 = k0 + a.K_each < a.K ? k0 + a.K_each : a.K;
    f32x4 acc[S::FP][S::FQ];
    product<T, FORM, TWO, ALIGNED, S, STAGES>(a, p0, q0, k0, k1, lds, acc);
    if constexpr (FORM != kWeightGrad && !GRAD) {
        if (a.sums) return put_sums<S>(a, FORM == kForward && TWO ? 2 : 1, p0, q0, split, acc);
    }
    epilogue<T, O, FORM, TWO, GRAD, S>(a, p0, q0, split, acc);
}

// Large products: workgroup b takes the places b, b + gridDim.x, ... of tile_of's order; gridDim.x is a multiple of eight, so its
// tiles stay on its XCD.  The next tile's first operands are asked for before this one's results are written.
template <typename T, typename O, int FORM, bool TWO, bool GRAD, typename S>
__global__ __launch_bounds__(S::kThreads, 2) void k_wide(const Args a, const unsigned places, const unsigned splits) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    struct Place { int64_t p0, q0, k0, k1, steps; unsigned split; };
    Stream<T, FORM, TWO, S> stream;
    Place now, next;
    unsigned b = blockIdx.x;
    auto find = [&](Place& at) {      // the next place that has a tile, its operands' addresses
        for (; b < places; b += gridDim.x) {
            unsigned tp, tq;
            if (!tile_of(a, splits, b, tp, tq, at.split)) continue;
            at.p0 = (int64_t)tp * (FORM == kForward && TWO ? S::kCols / 2 : S::kCols);
            at.q0 = (int64_t)tq * S::kRows;
            at.k0 = (int64_t)at.split * a.K_each;
            at.k1 = at.k0 + a.K_each < a.K ? at.k0 + a.K_each : a.K;
            at.steps = (at.k1 - at.k0) / Kind<T>::kStep;
            stream.begin(a, at.p0, at.q0, at.k0);
            b += gridDim.x;
            return true;
        }
        return false;
    };
    if (!find(next)) return;
    stream.ask_first(lds, next.steps);
    for (bool more = true; more;) {
        now = next;
        wait_loads<0>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        f32x4 acc[S::FP][S::FQ];
        stream.product(now.steps, lds, acc);
        const int64_t done = now.k0 + now.steps * Kind<T>::kStep;
        if (done < now.k1) stream.rest(a, now.p0, now.q0, done, now.k1, lds, acc);
        more = find(next);
        if (more) stream.ask_first(lds, next.steps);
        if constexpr (FORM != kWeightGrad && !GRAD) {
            if (a.sums) {
                put_sums<S>(a, FORM == kForward && TWO ? 2 : 1, now.p0, now.q0, now.split, acc);
                continue;
            }
        }
        epilogue<T, O, FORM, TWO, GRAD, S>(a, now.p0, now.q0, now.split, acc);
    }
}

// The splits' sums of a tile S, added in their order, and what becomes of them: two pieces of columns and one of rows of each wave to a workgroup.
template <typename S> struct Part {
    static constexpr int kThreads = S::kThreads, kUsed = 16, FP = 2, FQ = 1, kLast = S::kThreads / 64 - 1;
    static constexpr int kParts = S::FQ * S::FP / 2;
    static __device__ __forceinline__ int p_piece(int wave, int i) { return S::p_piece(wave, i); }
    static __device__ __forceinline__ int q_piece(int wave, int) { return S::q_piece(wave, 0); }
    static constexpr int kCols = (S::p_piece(kLast, 1) + 1) * 16, kRows = (S::q_piece(kLast, 0) + 1) * 16;      // what they span
};
template <typename T, typename O, int FORM, bool TWO, typename S>
__global__ __launch_bounds__(S::kThreads) void k_join(const Args a, const unsigned splits) {
    constexpr int kBy = FORM == kForward && TWO ? 2 : 1;
    const unsigned tile = blockIdx.x / Part<S>::kParts, part = blockIdx.x % Part<S>::kParts, j = part % S::FQ, i = part / S::FQ * 2;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t p0 = (int64_t)(tile % a.p_tiles) * (S::kCols / kBy) + S::p_piece(0, i) / kBy * 16, q0 = (int64_t)(tile / a.p_tiles) * S::kRows + S::q_piece(0, j) * 16;
    if (p0 + S::p_piece(wave, 0) / kBy * 16 >= a.p_count || q0 + S::q_piece(wave, 0) * 16 >= a.q_count) return;
    const bool both = p0 + S::p_piece(wave, 1) / kBy * 16 < a.p_count;
    const int64_t each = (int64_t)a.p_tiles * a.q_tiles * S::kThreads * (S::FP * S::FQ);
    const f32x4* from = a.sums + ((int64_t)tile * (S::kThreads / 64) + wave) * (S::FP * S::FQ * 64) + (i * S::FQ + j) * 64 + lane;
    const int second = both ? S::FQ * 64 : 0;
    f32x4 total[2][1] = {{f32x4{0.f, 0.f, 0.f, 0.f}}, {f32x4{0.f, 0.f, 0.f, 0.f}}};
#pragma unroll 4
    for (unsigned s = 0; s < splits; ++s) {
        const f32x4 x = from[s * each], y = from[s * each + second];
#pragma unroll
        for (int e = 0; e < 4; ++e) { total[0][0][e] += x[e]; total[1][0][e] += y[e]; }
    }
    epilogue<T, O, FORM, TWO, false, Part<S>>(a, p0, q0, 0, total);
}

// Products of few rows (up to 16 NQ): bound by the weights' bytes.  A workgroup has 16 columns of the result, its waves a share of the contraction each, operands go
// from memory to the matrix instructions without LDS, and the waves' sums are added in their order.  A wave asks for U steps of both operands at once;
// with 16 waves that is 100 to 200 KB in flight on a CU.
//   float32: v_mfma_f32_16x16x4_f32, products exact (a memory-bound kernel has no use for three parts)
//
// Where 16 columns and 16 rows a workgroup leave CUs without one, a workgroup has 16 / NS columns and as many rows: the 16 rows and columns of the matrix
// instruction are NS stretches of the contraction beside each other, and only the products of a stretch with itself, the blocks on its diagonal, count.
// x 4096 x 1024 bf16, us: one row 7.3 with 64 workgroups, 4.5 with 256; 7 rows 8.5 with 64, 6.1 with 128, 6.2 with 512; 16 rows 9.9 with 64, 6.5 with 256.
template <int BY, int NQ, int NS> struct FewShape {
    static constexpr int kCols = 16 * BY, kRows = 16 * NQ / NS, FP = BY, FQ = 1, kUsed = 16 / NS;
    static constexpr __host__ __device__ __forceinline__ int p_piece(int, int i) { return i; }
    static constexpr __host__ __device__ __forceinline__ int q_piece(int wave, int) { return wave; }
};
template <typename T, typename O, bool TWO, int NQ, int NS, bool ALIGNED>
__global__ __launch_bounds__(1024) void k_few(const Args a) {
    constexpr int BY = TWO ? 2 : 1, CE = 16 / (int)sizeof(T), U = NQ == 4 ? 2 : 4;
    using S = FewShape<BY, NQ, NS>;
    static_assert(NS == 1 || NQ == 1, "");
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6, g = lane >> 4;
    const int own = lane & (S::kUsed - 1), stretch = (lane & 15) / S::kUsed;
    const int64_t p0 = (int64_t)blockIdx.x * S::kUsed, q0 = (int64_t)blockIdx.y * S::kRows;      // (NS > 1: as many rows as columns)
    const int64_t pr = p0 + own < a.p_count ? p0 + own : a.p_count - 1;
    const T *W[BY], *X[NQ];
#pragma unroll
    for (int w = 0; w < BY; ++w) W[w] = reinterpret_cast<const T*>(a.P[w]) + pr * a.p_ld;
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
        const int64_t q = q0 + 16 * j + own < a.q_count ? q0 + 16 * j + own : a.q_count - 1;
        X[j] = reinterpret_cast<const T*>(a.Q) + q * a.q_ld;
    }
    constexpr int kAtOnce = 4 * CE * U;      // contraction indices that a wave asks for at once
    const int64_t each = (a.K + (int64_t)(waves * NS) * kAtOnce - 1) / ((int64_t)(waves * NS) * kAtOnce) * kAtOnce;
    const int64_t first = wave * NS * each, k0 = first + stretch * each, k1 = k0 + each < a.K ? k0 + each : a.K;
    f32x4 acc[BY][NQ];
#pragma unroll
    for (int w = 0; w < BY; ++w)
#pragma unroll
        for (int j = 0; j < NQ; ++j) acc[w][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int64_t done = 0; done < each && first + done < a.K; done += kAtOnce) {
        const int64_t k = k0 + done;
        u32x4 wv[BY][U], xv[NQ][U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t at = k + u * 4 * CE + g * CE;
#pragma unroll
            for (int w = 0; w < BY; ++w) wv[w][u] = part_of_row<T, ALIGNED>(W[w], at, k1, true);
#pragma unroll
            for (int j = 0; j < NQ; ++j) xv[j][u] = part_of_row<T, ALIGNED>(X[j], at, k1, true);
        }
#pragma unroll
        for (int w = 0; w < BY; ++w)
#pragma unroll
            for (int j = 0; j < NQ; ++j) {
                f32x4& c = acc[w][j];
                if constexpr (sizeof(T) == 1) {
#pragma unroll
                    for (int u = 0; u < U; u += 2) {
                        union { u32x4 h[2]; i32x8 v; } x, y;
                        x.h[0] = wv[w][u]; x.h[1] = wv[w][u + 1];
                        y.h[0] = xv[j][u]; y.h[1] = xv[j][u + 1];
                        c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x.v, y.v, c, 0, 0, 0, 0, 0, 0);
                    }
                } else if constexpr (sizeof(T) == 2) {
#pragma unroll
                    for (int u = 0; u < U; ++u) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, wv[w][u]), __builtin_bit_cast(bf16x8, xv[j][u]), c, 0, 0, 0);
                } else {
#pragma unroll
                    for (int u = 0; u < U; ++u)
#pragma unroll
                        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(wv[w][u][e]), __uint_as_float(xv[j][u][e]), c, 0, 0, 0);
                }
            }
    }
    f32x4* sums = reinterpret_cast<f32x4*>(lds);      // [waves][BY][NQ][64]
#pragma unroll
    for (int w = 0; w < BY; ++w)
#pragma unroll
        for (int j = 0; j < NQ; ++j) sums[((wave * BY + w) * NQ + j) * 64 + lane] = acc[w][j];
    __syncthreads();
    if (wave >= NQ) return;
    f32x4 total[BY][1];
#pragma unroll
    for (int w = 0; w < BY; ++w) {
        f32x4 t = sums[(w * NQ + wave) * 64 + lane];
        for (int v = 1; v < waves; ++v) {
            const f32x4 s = sums[((v * BY + w) * NQ + wave) * 64 + lane];
#pragma unroll
            for (int e = 0; e < 4; ++e) t[e] += s[e];
        }
        if constexpr (NS > 1) {      // to the first stretch's lanes
            f32x4 all = t;
#pragma unroll
            for (int n = 1; n < NS; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) all[e] += __shfl(t[e], (lane + n * (S::kUsed / 4 * 16 + S::kUsed)) & 63);
            t = all;
        }
        total[w][0] = t;
    }
    epilogue<T, O, kForward, TWO, false, S>(a, p0, q0, 0, total);
}

#if TGT_GATED_PART == 0
// Sums over the splits of a weight gradient, in their order, four elements a thread.  Elements from n_first on go to the second output.
template <typename O> __global__ __launch_bounds__(256) void k_add_splits(const float* __restrict__ partial, int splits, int64_t n, int64_t n_first, O* __restrict__ out0,
                                                                          O* __restrict__ out1) {
    const int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (e >= n) return;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (n % 4 == 0) {
#pragma unroll 4
        for (int w = 0; w < splits; ++w) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(partial + w * n + e);
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] += v[i];
        }
    } else {
        for (int w = 0; w < splits; ++w)
            for (int i = 0; i < 4; ++i)
                if (e + i < n) s[i] += partial[w * n + e + i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (e + i < n) from_float(e + i < n_first ? out0[e + i] : out1[e + i - n_first], s[i]);
}

// Column sums of a matrix of rows of M elements: workgroup (64 columns, share of the rows) -> partial[share][M].  Eight rows in flight a wave; bound by their
// latency where there are few columns.
template <typename O> __global__ __launch_bounds__(256) void k_column_sums(const O* __restrict__ x, int64_t N, int64_t M, int64_t rows_each, float* __restrict__ partial) {
    __shared__ float part[4][64];
    const int c = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t col = (int64_t)blockIdx.x * 64 + c, r0 = blockIdx.y * rows_each, r1 = r0 + rows_each < N ? r0 + rows_each : N;
    float s = 0.f;
    if (col < M) {
        int64_t r = r0 + w;
        for (; r + 28 < r1; r += 32) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = to_float(x[(r + 4 * i) * M + col]);
#pragma unroll
            for (int i = 0; i < 8; ++i) s += v[i];
        }
        for (; r < r1; r += 4) s += to_float(x[r * M + col]);
    }
    part[w][c] = s;
    __syncthreads();
    if (w == 0 && col < M) partial[blockIdx.y * M + col] = (part[0][c] + part[1][c]) + (part[2][c] + part[3][c]);
}

// dg = dh u act'(g), du = dh act(g) (one weight: du = dy act'(u)) from what the forward kept, a row of each weight side by side, and the column sums of what is
// written: workgroup (256 vectors: `across` of columns, so many rows side by side, share of the rows) -> partial[share][TWO ? 2 F : F] (null: not wanted).  Bound by
// memory: 16384 x 4096 bf16, 671 MB in 152 us.  WHOLE: rows of whole vectors, aligned.
template <typename O, int VE> struct KeptPiece {      // as it is in memory until it is used
    uint2 p[VE / 4];
    template <bool WHOLE> __device__ __forceinline__ void read(const O* from, int) {
        if constexpr (WHOLE && VE == 8) {
            const u32x4 v = *reinterpret_cast<const u32x4*>(from);
            p[0] = make_uint2(v.x, v.y);
            p[VE / 4 - 1] = make_uint2(v.z, v.w);
        } else p[0] = *reinterpret_cast<const uint2*>(from);
    }
    __device__ __forceinline__ void values(float (&v)[VE]) const {
#pragma unroll
        for (int i = 0; i < VE / 4; ++i) {
            float f[4];
            unpack_four(p[i], f);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[i * 4 + e] = f[e];
        }
    }
};
template <> struct KeptPiece<float, 4> {
    Four<float> f;
    template <bool WHOLE> __device__ __forceinline__ void read(const float* from, int n) { f = load4<float, WHOLE>(from, n); }
    __device__ __forceinline__ void values(float (&v)[4]) const {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = f.e[e];
    }
};
template <typename O, bool TWO, int ACT, int VE, bool WHOLE>
__global__ __launch_bounds__(256) void k_kept_grad(const O* __restrict__ kept, const O* __restrict__ dy, int64_t N, int64_t F, int64_t rows_each, int across,
                                                   O* __restrict__ du, float* __restrict__ partial) {
    constexpr int NW = TWO ? 2 : 1, U = 4;      // rows in flight
    constexpr bool EXACT = sizeof(O) == 4;
    static_assert(VE == 4 || WHOLE, "");
    struct alignas(VE * sizeof(O)) Some { O e[VE]; };
    __shared__ float side[256 * VE];
    const int tx = threadIdx.x & (across - 1), ty = threadIdx.x / across, beside = 256 / across;
    const int64_t c = ((int64_t)blockIdx.x * across + tx) * VE, r0 = blockIdx.y * rows_each, r1 = r0 + rows_each < N ? r0 + rows_each : N, width = kept_width<O>(F);
    const int left = c >= F ? 0 : WHOLE || F - c >= VE ? VE : (int)(F - c);
    float sums[NW][VE];
#pragma unroll
    for (int w = 0; w < NW; ++w)
#pragma unroll
        for (int e = 0; e < VE; ++e) sums[w][e] = 0.f;
    for (int64_t r = r0 + ty; r < r1 && left; r += U * beside) {
        const int n = (r1 - r + beside - 1) / beside < U ? (int)((r1 - r + beside - 1) / beside) : U;
        struct { KeptPiece<O, VE> k[NW]; Some dy; } in[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int64_t row = i < n ? r + i * beside : r;
#pragma unroll
            for (int w = 0; w < NW; ++w) in[i].k[w].template read<WHOLE>(kept + (row * NW + w) * width + c, left);
            if constexpr (WHOLE) in[i].dy = *reinterpret_cast<const Some*>(dy + row * F + c);
            else {
                const Four<O> f = load4<O, false>(dy + row * F + c, left);
#pragma unroll
                for (int e = 0; e < VE; ++e) in[i].dy.e[e] = f.e[e];
            }
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
            if (i >= n) break;
            Some out[NW];
            float k[NW][VE];
#pragma unroll
            for (int w = 0; w < NW; ++w) in[i].k[w].values(k[w]);
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const float g = k[0][e], d = to_float(in[i].dy.e[e]);
                float o[NW];
                if constexpr (TWO) {
                    float f, s;
                    act_and_slope<EXACT, ACT>(g, f, s);
                    o[0] = d * k[NW - 1][e] * s;
                    o[NW - 1] = d * f;
                } else o[0] = slope_of<EXACT, ACT>(g, d);
#pragma unroll
                for (int w = 0; w < NW; ++w) {
                    sums[w][e] += o[w];
                    from_float(out[w].e[e], o[w]);
                }
            }
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                O* to = du + ((r + i * beside) * NW + w) * F + c;
                if constexpr (WHOLE) *reinterpret_cast<Some*>(to) = out[w];
                else {
#pragma unroll
                    for (int e = 0; e < VE; ++e)
                        if (e < left) to[e] = out[w].e[e];
                }
            }
        }
    }
    if (!partial) return;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        if (beside > 1) {      // the rows side by side, in their order
            __syncthreads();
#pragma unroll
            for (int e = 0; e < VE; ++e) side[e * 256 + threadIdx.x] = sums[w][e];
            __syncthreads();
            if (ty) continue;
#pragma unroll
            for (int e = 0; e < VE; ++e)
                for (int k = 1; k < beside; ++k) sums[w][e] += side[e * 256 + k * across + tx];
        }
#pragma unroll
        for (int e = 0; e < VE; ++e)
            if (e < left) partial[((int64_t)blockIdx.y * NW + w) * F + c + e] = sums[w][e];
    }
}
int across_of(int64_t F, int VE) {
    int n = 1;
    while (n < 256 && n * VE < F) n *= 2;
    return n;
}
template <typename O, bool TWO, int VE, bool WHOLE> void launch_kept_grad_as(const void* kept, const void* dy, int64_t N, int64_t F, int64_t rows_each, int shares, int act, void* du, float* partial, hipStream_t st) {
    const int across = across_of(F, VE);
    const dim3 grid((unsigned)((F + across * VE - 1) / (across * VE)), (unsigned)shares);
#define X(ACT) hipLaunchKernelGGL((k_kept_grad<O, TWO, ACT, VE, WHOLE>), grid, dim3(256), 0, st, (const O*)kept, (const O*)dy, N, F, rows_each, across, (O*)du, partial)
    switch (act) {
        case TGT_ACT_SILU: X(TGT_ACT_SILU); break;
        case TGT_ACT_GELU: X(TGT_ACT_GELU); break;
        case TGT_ACT_RELU: X(TGT_ACT_RELU); break;
        default: X(TGT_ACT_NONE); break;
    }
#undef X
}
template <typename O> void launch_kept_grad(const void* kept, const void* dy, int n, int64_t N, int64_t F, int64_t rows_each, int shares, int act, void* du, float* partial, hipStream_t st) {
    constexpr int VE = 16 / (int)sizeof(O);
    const bool whole = F % VE == 0 && (((uintptr_t)dy | (uintptr_t)du) & 15) == 0;
    if (n == 2) return whole ? launch_kept_grad_as<O, true, VE, true>(kept, dy, N, F, rows_each, shares, act, du, partial, st) : launch_kept_grad_as<O, true, 4, false>(kept, dy, N, F, rows_each, shares, act, du, partial, st);
    return whole ? launch_kept_grad_as<O, false, VE, true>(kept, dy, N, F, rows_each, shares, act, du, partial, st) : launch_kept_grad_as<O, false, 4, false>(kept, dy, N, F, rows_each, shares, act, du, partial, st);
}

__global__ __launch_bounds__(256) void k_zero(uint16_t* __restrict__ p, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = 0;
}
#endif

using Square = Shape<128, 128, 2, 2>;

template <typename T, typename O, int FORM, bool TWO, typename S> int join(const Args& a, int splits, hipStream_t st) {
    if (!a.sums) return TGT_OK;
    hipLaunchKernelGGL((k_join<T, O, FORM, TWO, S>), dim3(a.p_tiles * a.q_tiles * Part<S>::kParts), dim3(S::kThreads), 0, st, a, (unsigned)splits);
    TGT_HIP_CHECK(hipGetLastError());
    return TGT_OK;
}

template <typename T, typename O, int FORM, bool TWO, bool GRAD, bool ALIGNED, typename S, int STAGES>
int launch(Args a, int splits, hipStream_t st) {
    constexpr int kCols = FORM == kForward && TWO ? S::kCols / 2 : S::kCols;
    a.p_tiles = (unsigned)((a.p_count + kCols - 1) / kCols);
    a.q_tiles = (unsigned)((a.q_count + S::kRows - 1) / S::kRows);
    const int64_t tiles = (int64_t)a.p_tiles * a.q_tiles * splits;
    if (tiles > (1ll << 30)) { set_error("torchgt: a product of more than 2^30 tiles"); return TGT_ERR_UNSUPPORTED; }
    constexpr int kLds = STAGES * (S::kCols + S::kRows) * Kind<T>::kRowBytes * Kind<T>::kPlanes;
    auto* kernel = k_product<T, O, FORM, TWO, GRAD, ALIGNED, S, STAGES>;
    if (kLds > 65536) {
        static std::atomic<uint64_t> done{0};
        const int rc = allow_lds((const void*)kernel, kLds, done);
        if (rc != TGT_OK) return rc;
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)((tiles + 7) / 8 * 8)), dim3(S::kThreads), kLds, st, a, (unsigned)splits);
    TGT_HIP_CHECK(hipGetLastError());
    if constexpr (FORM != kWeightGrad && !GRAD) return join<T, O, FORM, TWO, S>(a, splits, st);
    return TGT_OK;
}

template <typename T, typename O, int FORM, bool TWO, bool GRAD, typename S>
int launch_wide(Args a, int splits, hipStream_t st) {
    constexpr int kCols = FORM == kForward && TWO ? S::kCols / 2 : S::kCols;
    a.p_tiles = (unsigned)((a.p_count + kCols - 1) / kCols);
    a.q_tiles = (unsigned)((a.q_count + S::kRows - 1) / S::kRows);
    const int64_t places = ((int64_t)a.p_tiles * a.q_tiles * splits + 7) / 8 * 8;
    if (places > (1ll << 30)) { set_error("torchgt: a product of more than 2^30 tiles"); return TGT_ERR_UNSUPPORTED; }
    auto* kernel = k_wide<T, O, FORM, TWO, GRAD, S>;
    static std::atomic<uint64_t> done{0};
    const int rc = allow_lds((const void*)kernel, S::kLds, done);
    if (rc != TGT_OK) return rc;
    const unsigned grid = (unsigned)std::min<int64_t>(places, num_cus() / 8 * 8);
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(S::kThreads), S::kLds, st, a, (unsigned)places, (unsigned)splits);
    TGT_HIP_CHECK(hipGetLastError());
    if constexpr (FORM != kWeightGrad && !GRAD) return join<T, O, FORM, TWO, S>(a, splits, st);
    return TGT_OK;
}

template <typename T, typename O, bool TWO, int NQ, int NS, bool ALIGNED> int launch_few(const Args& a, hipStream_t st) {
    constexpr int kBy = TWO ? 2 : 1, kAtOnce = 4 * (16 / (int)sizeof(T)) * (NQ == 4 ? 2 : 4) * NS;
    // halves of the columns while CUs are left without a workgroup and four waves have something to do
    if constexpr (NQ == 1 && NS < 4) {
        if ((a.p_count * 2 * NS + 15) / 16 * ((a.q_count * 2 * NS + 15) / 16) <= num_cus() && a.K >= 8 * kAtOnce) return launch_few<T, O, TWO, NQ, 2 * NS, ALIGNED>(a, st);
    }
    // a share of the contraction for each wave, 4 (16 rows for each: so many lanes that add up) to 16 waves
    const int waves = (int)std::max<int64_t>(4, std::min<int64_t>(16, (a.K + kAtOnce - 1) / kAtOnce));
    const int bytes = waves * kBy * NQ * 64 * 16;      // at most 128 KB
    auto* kernel = k_few<T, O, TWO, NQ, NS, ALIGNED>;
    if (16 * kBy * NQ * 64 * 16 > 65536) {
        static std::atomic<uint64_t> done{0};
        const int rc = allow_lds((const void*)kernel, 16 * kBy * NQ * 64 * 16, done);
        if (rc != TGT_OK) return rc;
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)((a.p_count + 16 / NS - 1) / (16 / NS)), (unsigned)((a.q_count * NS + 16 * NQ - 1) / (16 * NQ))), dim3(64 * waves), bytes, st, a);
    TGT_HIP_CHECK(hipGetLastError());
    return TGT_OK;
}
// How a product is cut: tiles of 128 x 128 (halves 0) or 256 rows x 128 or 256 columns (kernels for 16- and 8-bit operands, aligned rows that 32-bit offsets
// reach, K >= 256), and splits of the contraction where there are fewer tiles than CUs, whose sums are joined by a kernel of their own.  What is taken is what
// takes least by this account, in us, fitted to measurements of each kernel at K 256 to 8192 and 64 to 1024 tiles:
struct Way { int halves, splits; int64_t K_each, bytes; };
template <typename T> Way way_of(int64_t p_count, int64_t q_count, int64_t K, int by, bool wide, bool cut) {
    constexpr int kSize = sizeof(T);
    static constexpr double kFixed[3] = {kSize == 4 ? 4. : 5., 8.5, 14.}, kStep[3] = {kSize == 4 ? 2.8 : kSize == 2 ? 1.2 : 1.1, .85, 1.44};
    const int64_t cus = num_cus(), steps = (K + Kind<T>::kStep - 1) / Kind<T>::kStep;
    Way best{};
    double least = 1e300;
    for (int h = 0; h <= (wide ? kSize == 1 ? 1 : 2 : 0); ++h) {      // (8-bit operands beside 128 sums: no registers, and reloads from scratch wait for all loads)
        const int64_t cols = (h == 2 ? 256 : 128) / by, rows = h ? 256 : 128, tiles = (p_count + cols - 1) / cols * ((q_count + rows - 1) / rows);
        const int64_t slots = h ? cus : 2 * cus, most = cut && h < 2 ? std::min(slots / tiles, steps / 2) : 1;      // (two workgroups of the small tiles to a CU, a third slower each)
        for (int64_t s = 1;; s = std::min(most, s + (s + 1) / 2)) {      // (a dozen of them: this runs on the host in every call)
            const int64_t each = (steps + s - 1) / s, bytes = s > 1 ? s * tiles * rows * 128 * 4 : 0;
            const double us = (tiles * s + slots - 1) / slots * (kFixed[h] + each * kStep[h] * (tiles * s > cus && !h ? 1.3 : 1.)) + (s > 1 ? 4. + bytes * .4e-6 : 0.);
            if (us < least && (steps + each - 1) / each == s) { least = us; best = Way{h, (int)s, each * Kind<T>::kStep, bytes}; }
            if (s >= most) break;
        }
    }
    return best;
}
bool wide_rows(const Args& a) { return a.K >= 256 && a.p_ld < (1 << 21) && a.q_ld < (1 << 21); }
bool aligned16(const void* p, int64_t ld, int size) { return ((uintptr_t)p & 15) == 0 && ld * size % 16 == 0; }

}  // namespace

// One product in the form asked for; TWO: a.P[1] is given
struct Room { void* p; int64_t bytes; };      // for the sums of splits
// Whether a product is one of few rows: up to 64 of them, or not even a workgroup of 16 rows and 16 columns for every CU (us, kernel of few rows / tiles and
// joined sums: 64 x 4096 x 1024 bf16 10.5 / 13.6, float32 18.3 / 23.8; 64 x 1024 x 4096 8.1 / 13.2; 65 x 1024 x 256 5.3 / 9.3)
static inline bool few_rows(int64_t q_count, int64_t p_count) { return q_count <= 64 || (q_count + 15) / 16 * ((p_count + 15) / 16) <= num_cus(); }
template <typename T, typename O> int product_forward(Args a, bool grad, Room room, hipStream_t st);
template <typename T> int product_input_grad(Args a, Room room, hipStream_t st);
template <typename T> int product_weight_grad(Args a, int& splits, hipStream_t st);      // (more than one split: to a.partial)

// Bytes that the sums of splits take, whatever the operands' alignment
template <typename T> int64_t room_of(int64_t p_count, int64_t q_count, int64_t K, int by) {
    return std::max(way_of<T>(p_count, q_count, K, by, false, true).bytes, way_of<T>(p_count, q_count, K, by, sizeof(T) < 4 && K >= 256, true).bytes);
}

#if TGT_GATED_PART > 0
int take(Args& a, const Way& way, const Room& room) {
    a.K_each = way.K_each;
    if (!way.bytes) return TGT_OK;
    if (!room.p || room.bytes < way.bytes || ((uintptr_t)room.p & 15)) {
        set_error("torchgt: a product's workspace of %lld bytes (16-byte aligned) needed, got %lld", (long long)way.bytes, (long long)room.bytes);
        return TGT_ERR_WORKSPACE;
    }
    a.sums = reinterpret_cast<f32x4*>(room.p);
    return TGT_OK;
}
template <typename T, typename O> int product_forward(Args a, bool grad, Room room, hipStream_t st) {
    constexpr int kStages = sizeof(T) == 4 ? 1 : 2;
    const bool two = a.P[1] != nullptr;
    const bool al = aligned16(a.Q, a.q_ld, sizeof(T)) && aligned16(a.P[0], a.p_ld, sizeof(T)) && (!two || aligned16(a.P[1], a.p_ld, sizeof(T)));
    if (!grad && few_rows(a.q_count, a.p_count)) {
        // more rows to a workgroup only where there is one for every CU: they share its reads of the weights, but a workgroup takes longer by 3 us for 16 rows of 4096
        // (64 x 4096 x 1024 bf16, us: 16 rows each 10.5, all 64 20.8)
        const int64_t blocks = (a.p_count + 15) / 16, sixteens = (a.q_count + 15) / 16;
        const int nq = blocks * sixteens <= num_cus() ? 1 : blocks * ((sixteens + 1) / 2) <= num_cus() || sixteens <= 2 ? 2 : 4;
#define X(TWO, NQ, AL) if (two == TWO && (nq == NQ || (NQ == 1 && sixteens == 1)) && al == AL) return launch_few<T, O, TWO, NQ, 1, AL>(a, st)
        X(false, 1, true); X(true, 1, true); X(false, 2, true); X(true, 2, true); X(false, 4, true); X(true, 4, true);
        X(false, 1, false); X(true, 1, false); X(false, 2, false); X(true, 2, false); X(false, 4, false); X(true, 4, false);
#undef X
    }
    const Way way = way_of<T>(a.p_count, a.q_count, a.K, two ? 2 : 1, sizeof(T) < 4 && al && wide_rows(a), !grad);
    if (const int rc = take(a, way, room)) return rc;
    if constexpr (sizeof(T) < 4) {
#define X(TWO, GRAD, PH) if (two == TWO && grad == GRAD && way.halves == PH) return launch_wide<T, O, kForward, TWO, GRAD, Wide<PH>>(a, way.splits, st)
        X(false, false, 1); X(true, false, 1);
        if constexpr (sizeof(T) > 1) { X(false, false, 2); X(true, false, 2); X(false, true, 1); X(true, true, 1); X(false, true, 2); X(true, true, 2); }
#undef X
    }
#define X(TWO, GRAD, AL) if (two == TWO && grad == GRAD && al == AL) return launch<T, O, kForward, TWO, GRAD, AL, Square, kStages>(a, way.splits, st)
    X(false, false, true); X(true, false, true); X(false, false, false); X(true, false, false);
    if constexpr (sizeof(T) > 1) { X(false, true, true); X(true, true, true); X(false, true, false); X(true, true, false); }
#undef X
    return TGT_ERR_INVALID_ARG;
}
#endif
#if TGT_GATED_PART == 1 || TGT_GATED_PART == 2
template <typename T> int product_input_grad(Args a, Room room, hipStream_t st) {
    constexpr int kStages = sizeof(T) == 4 ? 1 : 2;
    const bool two = a.P[1] != nullptr;
    const bool al = aligned16(a.Q, a.q_ld, sizeof(T)) && aligned16(a.P[0], a.p_ld, sizeof(T)) && (!two || aligned16(a.P[1], a.p_ld, sizeof(T)));
    const Way way = way_of<T>(a.p_count, a.q_count, a.K, 1, sizeof(T) < 4 && al && wide_rows(a) && a.p_count % 8 == 0 && (!two || a.K_first % Kind<T>::kStep == 0), true);
    if (const int rc = take(a, way, room)) return rc;
    if constexpr (sizeof(T) < 4) {
#define X(TWO, PH) if (two == TWO && way.halves == PH) return launch_wide<T, T, kInputGrad, TWO, false, Wide<PH>>(a, way.splits, st)
        X(false, 1); X(true, 1); X(false, 2); X(true, 2);
#undef X
    }
#define X(TWO, AL) if (two == TWO && al == AL) return launch<T, T, kInputGrad, TWO, false, AL, Square, kStages>(a, way.splits, st)
    X(false, true); X(true, true); X(false, false); X(true, false);
#undef X
    return TGT_ERR_INVALID_ARG;
}
template <typename T> int product_weight_grad(Args a, int& splits, hipStream_t st) {
    constexpr int kStages = sizeof(T) == 4 ? 1 : 2;
    const bool al = aligned16(a.Q, a.q_ld, sizeof(T)) && aligned16(a.P[0], a.p_ld, sizeof(T));
    const Way way = way_of<T>(a.p_count, a.q_count, a.K, 1, sizeof(T) < 4 && al && wide_rows(a) && a.p_count % 8 == 0 && a.q_count % 8 == 0, true);
    splits = way.splits;
    a.K_each = way.K_each;
    if (way.splits == 1) a.partial = nullptr;
    if constexpr (sizeof(T) < 4) {
        if (way.halves == 2) return launch_wide<T, T, kWeightGrad, false, false, Wide<2>>(a, way.splits, st);
        if (way.halves == 1) return launch_wide<T, T, kWeightGrad, false, false, Wide<1>>(a, way.splits, st);
    }
    if (al) return launch<T, T, kWeightGrad, false, false, true, Square, kStages>(a, way.splits, st);
    return launch<T, T, kWeightGrad, false, false, false, Square, kStages>(a, way.splits, st);
}
#endif
#if TGT_GATED_PART == 1
template int product_forward<b16, b16>(Args, bool, Room, hipStream_t);
template int product_input_grad<b16>(Args, Room, hipStream_t);
template int product_weight_grad<b16>(Args, int&, hipStream_t);
#elif TGT_GATED_PART == 2
template int product_forward<float, float>(Args, bool, Room, hipStream_t);
template int product_input_grad<float>(Args, Room, hipStream_t);
template int product_weight_grad<float>(Args, int&, hipStream_t);
#elif TGT_GATED_PART == 3
template int product_forward<e4m3, b16>(Args, bool, Room, hipStream_t);
template int product_forward<e4m3, float>(Args, bool, Room, hipStream_t);
#else

namespace {

// What the entry points share: n weights [F, K] (two: gate and up)
struct Call {
    const char* who;
    const void *x, *W[2], *b[2];
    int n;
    int64_t N;
    int K, F, dtype, act;
};

int check_call(const Call& c, int64_t most_rows = 0x7fffffff) {
    if (c.N < 0 || c.K < 1 || c.F < 1 || (c.dtype != TGT_DTYPE_F32 && c.dtype != TGT_DTYPE_BF16)) {
        set_error("%s: bad size or dtype", c.who);
        return TGT_ERR_INVALID_ARG;
    }
    if (c.N > most_rows || c.F > (1 << 24) || c.K > (1 << 24)) {
        set_error("%s: %lld rows of %d and %d features: at most 2^31 - 1 rows and 2^24 features", c.who, (long long)c.N, c.K, c.F);
        return TGT_ERR_UNSUPPORTED;
    }
    if (c.act != TGT_ACT_NONE && c.act != TGT_ACT_GELU && c.act != TGT_ACT_RELU && c.act != TGT_ACT_SILU) {
        set_error("%s: unknown activation %d", c.who, c.act);
        return TGT_ERR_INVALID_ARG;
    }
    if (c.N > 0 && (!c.x || !c.W[0] || (c.n == 2 && !c.W[1]))) {
        set_error("%s: null pointer", c.who);
        return TGT_ERR_INVALID_ARG;
    }
    return TGT_OK;
}

Args forward_args(const Call& c) {
    Args a{};
    a.P[0] = c.W[0]; a.P[1] = c.n == 2 ? c.W[1] : nullptr;
    a.Q = c.x;
    a.p_ld = a.q_ld = c.K;
    a.p_count = c.F; a.q_count = c.N;
    a.K = a.K_first = a.K_each = c.K;
    a.bias[0] = c.b[0]; a.bias[1] = c.n == 2 ? c.b[1] : nullptr;
    a.out_ld = c.F;
    a.act = c.act;
    return a;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
bool needs_du(int n, int act) { return n == 2 || act != TGT_ACT_NONE; }      // (else dy is the operand itself)
int in16(int dtype) { return dtype == TGT_DTYPE_F32 ? 4 : 8; }      // elements in 16 bytes
// Whether the kernels for small widths (gated_tiles.hip, linear_tiles.hip) are the faster ones; forward and backward kernels in us, those / the tiles of 128 and
// 256 rows, nodes x K x F, n weights:
//   bfloat16   one, no activation   500 x 128 x 128 19 / 33    2000 x 256 x 256 27 / 39    500 x 512 x 512 42 / 33    2000 x 512 x 512 45 / 50    8000 x 256 x 1024 70 / 55
//                                   32000 x 256 x 256 59 / 48
//              two                  2000 x 128 x 128 33 / 49   2000 x 256 x 256 56 / 60    500 x 64 x 1024 64 / 47    2000 x 512 x 512 97 / 68
//   float32    one, no activation   2000 x 256 x 256 40 / 60   500 x 512 x 512 64 / 49     2000 x 512 x 512 72 / 89    8000 x 512 x 512 123 / 150
//              two                  2000 x 64 x 64 31 / 69     500 x 256 x 256 83 / 65     8000 x 256 x 256 115 / 117  32000 x 64 x 1024 347 / 564   8000 x 512 x 512 294 / 255
// and a long contraction is not formed again where it can be kept (gelu, 2000 x 1024 x 64: bfloat16 60 / 47, float32 105 / 70; 32000: 178 / 282)
bool narrow(const Call& c) {
    const bool f32 = c.dtype == TGT_DTYPE_F32;
    const int64_t values = (int64_t)c.K * c.F * c.n;
    if (values > (f32 && c.N >= (needs_du(c.n, c.act) ? 4096 : 1024) ? 1 << 18 : 1 << 16) || (double)c.N * values > (f32 ? 8.6e9 : 1.6e9)) return false;
    if (needs_du(c.n, c.act) && c.K >= 512 && (!f32 || c.N < 16384)) return false;
    return c.K % in16(c.dtype) == 0 && aligned16(c.x) && aligned16(c.W[0]) && aligned16(c.W[1]);
}
NarrowArgs narrow_args(const Call& c, const void* more) {
    NarrowArgs a{};
    a.x = c.x; a.more = more;
    for (int w = 0; w < c.n; ++w) { a.W[w] = c.W[w]; a.bias[w] = c.b[w]; }
    a.N = c.N; a.K = c.K; a.F = a.out_ld = c.F; a.act = c.act;
    return a;
}

// What a forward that will have a backward is asked to keep: the products themselves, where forming them again takes longer than writing and reading them
// (16384 x K x 4096 gated bf16, us: the product again with the gradients behind it, K 1024 360; kept values read 155, written 45 more in the forward; a
// product takes about 0.3 us a K here, so 512 is where both take the same; float32 0.9 us a K and twice the bytes, three parts' products: 128).
bool keeps(const Call& c) { return needs_du(c.n, c.act) && c.N > 64 && !narrow(c) && c.K >= (c.dtype == TGT_DTYPE_F32 ? 128 : 512); }

int forward(const Call& c, const void* residual, void* out, void* kept, Room room, hipStream_t st) {
    int rc = check_call(c);
    if (rc != TGT_OK || c.N == 0) return rc;
    if (!out) { set_error("%s: null pointer", c.who); return TGT_ERR_INVALID_ARG; }
    if (!aligned16(kept)) { set_error("%s: what is kept has to start on 16 bytes", c.who); return TGT_ERR_INVALID_ARG; }
    if (!few_rows(c.N, c.F) && narrow(c) && !kept) {
        NarrowArgs a = narrow_args(c, residual);
        a.out[0] = out;
        KernelTimer t(KS_LINEAR_FWD, st);
        return gated_tiles(a, false, c.dtype, st);
    }
    Args a = forward_args(c);
    a.residual = residual;
    a.out[0] = out;
    a.kept = kept;
    KernelTimer t(KS_LINEAR_FWD, st);
    return c.dtype == TGT_DTYPE_F32 ? product_forward<float, float>(a, false, room, st) : product_forward<b16, b16>(a, false, room, st);
}

int forward_8bit(const Call& c, const float* x_scales, const float* s0, const float* s1, const void* residual, void* out, Room room, hipStream_t st) {
    int rc = check_call(c);
    if (rc != TGT_OK) return rc;
    if (c.K % 16) {
        set_error("%s: %d features: operands in 8 bits need a multiple of 16", c.who, c.K);
        return TGT_ERR_UNSUPPORTED;
    }
    if (c.N == 0) return TGT_OK;
    if (!out || !x_scales || !s0 || (c.n == 2 && !s1)) { set_error("%s: null pointer", c.who); return TGT_ERR_INVALID_ARG; }
    Args a = forward_args(c);
    a.q_scale = x_scales;
    a.p_scale[0] = s0; a.p_scale[1] = s1;
    a.residual = residual;
    a.out[0] = out;
    KernelTimer t(KS_LINEAR_FWD, st);
    return c.dtype == TGT_DTYPE_F32 ? product_forward<e4m3, float>(a, false, room, st) : product_forward<e4m3, b16>(a, false, room, st);
}

// How the backward lays out its workspace, and how it cuts the nodes
struct Plan {
    int64_t du_bytes, between, bytes, rows_each;
    int shares, kept_shares;
};
int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }
Plan plan_of(int n, int64_t N, int K, int F, int dtype, int act) {
    Plan p{};
    const int64_t size = dtype == TGT_DTYPE_F32 ? 4 : 2, cols = (int64_t)n * F;
    p.du_bytes = n == 2 || act != TGT_ACT_NONE ? up16(N * cols * size) : 0;      // (without an activation dy is the operand itself)
    p.shares = (int)std::max<int64_t>(1, std::min<int64_t>(512, (N + 31) / 32));
    p.rows_each = (N + p.shares - 1) / p.shares;
    const int beside = 256 / across_of(F, in16(dtype));
    p.kept_shares = (int)std::max<int64_t>(1, std::min<int64_t>(512, (N + 8 * beside - 1) / (8 * beside)));      // (their rows are in flight together: latency counts before bandwidth)
    // one after the other: the sums of dx's splits, those of the weights' gradients (no more than their whole tiles would take)
    p.between = up16(dtype == TGT_DTYPE_F32 ? std::max(room_of<float>(K, N, cols, 1), room_of<float>(K, cols, N, 1)) : std::max(room_of<b16>(K, N, cols, 1), room_of<b16>(K, cols, N, 1)));
    p.bytes = p.du_bytes + p.between + up16((int64_t)p.kept_shares * cols * 4);
    return p;
}

int64_t workspace_bytes_of(int n, int64_t N, int K, int F, int dtype, int act);

// The backward where the widths are small: one kernel for dg and du, rows of 16 bytes, then the linears' own backward of two weights of one shape (which reads them
// once for dx and once for all weight and bias gradients)
int padded_width(int F, int dtype) { return (F + in16(dtype) - 1) / in16(dtype) * in16(dtype); }
int64_t narrow_bytes(int n, int64_t N, int K, int F, int dtype, int act) {
    const int64_t Fp = padded_width(F, dtype), size = dtype == TGT_DTYPE_F32 ? 4 : 2;
    return (needs_du(n, act) ? n * up16(N * Fp * size) : 0) + (Fp != F ? up16(Fp * K * size) : 0) + up16(tgt_linear_bwd_workspace_bytes(n, K, (int)Fp));
}
int backward_narrow(const Call& c, const void* dy, void* dx, void* const* dW, void* const* db, char* ws, hipStream_t st) {
    const int Fp = padded_width(c.F, c.dtype);
    const bool f32 = c.dtype == TGT_DTYPE_F32;
    const int64_t size = f32 ? 4 : 2;
    const void *du[2] = {dy, nullptr}, *W[2] = {c.W[0], c.W[1]};
    if (needs_du(c.n, c.act)) {
        NarrowArgs a = narrow_args(c, dy);
        for (int w = 0; w < c.n; ++w) { du[w] = a.out[w] = ws; ws += up16(c.N * Fp * size); }
        a.out_ld = Fp;
        if (Fp != c.F) {      // (one weight: its rows behind the last are zeros for dx, their gradients are not wanted)
            W[0] = a.padded = ws;
            ws += up16((int64_t)Fp * c.K * size);
        }
        KernelTimer t(KS_LINEAR_FWD, st);
        if (const int rc = gated_tiles(a, true, c.dtype, st)) return rc;
    }
    const bool want_w = dW && dW[0], want_b = db && (db[0] || (c.n == 2 && db[1]));
    const int64_t bytes = tgt_linear_bwd_workspace_bytes(c.n, c.K, Fp);
    if (!want_w && !want_b) return dx ? tgt_linear_bwd(c.x, W, du, c.n, c.N, c.K, Fp, c.dtype, dx, nullptr, nullptr, nullptr, 0, st) : TGT_OK;
    tgt_reduce_desc r{};
    void* any[2] = {ws, ws};      // (where the sums go is said below)
    const int rc = tgt_linear_bwd_deferred(c.x, W, du, c.n, c.N, c.K, Fp, c.dtype, dx, any, any, ws, bytes, st, &r);
    if (rc != TGT_OK) return rc;
    const int each = Fp * c.K + Fp;
    r.n_out = 0;
    for (int w = 0; w < c.n; ++w) {
        const auto put = [&](void* out, int begin) { r.out[r.n_out] = out; r.begin[r.n_out++] = w * each + begin; };
        put(want_w ? dW[w] : nullptr, 0);
        if (Fp != c.F) put(nullptr, c.F * c.K);
        put(want_b ? db[w] : nullptr, Fp * c.K);
        if (Fp != c.F) put(nullptr, Fp * c.K + c.F);
    }
    return reduce_partials(&r, 1, c.dtype, st);
}
// Two weights of odd widths would need their rows padded too, and a gradient of odd rows that is the operand itself cannot be: those go the general way
bool narrow_backward(const Call& c, const void* dy) {
    return narrow(c) && (padded_width(c.F, c.dtype) == c.F || (c.n == 1 && c.act != TGT_ACT_NONE)) && (needs_du(c.n, c.act) || aligned16(dy));
}

int backward(const Call& c, const void* kept, const void* dy, void* dx, void* const* dW, void* const* db, void* workspace, int64_t workspace_bytes, hipStream_t st) {
    int rc = check_call(c);
    if (rc != TGT_OK) return rc;
    const bool f32 = c.dtype == TGT_DTYPE_F32;
    const int64_t size = f32 ? 4 : 2, cols = (int64_t)c.n * c.F;
    const bool want_w = dW && dW[0], want_b = db && (db[0] || (c.n == 2 && db[1]));
    if (want_w && c.n == 2 && !dW[1]) { set_error("%s: both weights' gradients or none", c.who); return TGT_ERR_INVALID_ARG; }
    if (c.N == 0) {      // nothing to add up
        for (int w = 0; w < c.n; ++w) {
            const int64_t m = (int64_t)c.F * c.K * (size / 2), v = c.F * (size / 2);
            if (want_w) hipLaunchKernelGGL(k_zero, dim3((unsigned)std::min<int64_t>((m + 255) / 256, 4096)), dim3(256), 0, st, (uint16_t*)dW[w], m);
            if (want_b && db[w]) hipLaunchKernelGGL(k_zero, dim3((unsigned)std::min<int64_t>((v + 255) / 256, 4096)), dim3(256), 0, st, (uint16_t*)db[w], v);
        }
        TGT_HIP_CHECK(hipGetLastError());
        return TGT_OK;
    }
    if (!dy) { set_error("%s: null pointer", c.who); return TGT_ERR_INVALID_ARG; }
    if (!aligned16(kept)) { set_error("%s: what is kept has to start on 16 bytes", c.who); return TGT_ERR_INVALID_ARG; }
    const Plan p = plan_of(c.n, c.N, c.K, c.F, c.dtype, c.act);
    const int64_t need = workspace_bytes_of(c.n, c.N, c.K, c.F, c.dtype, c.act);
    if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)) {
        set_error("%s: workspace of %lld bytes (16-byte aligned) needed, got %lld", c.who, (long long)need, (long long)workspace_bytes);
        return TGT_ERR_WORKSPACE;
    }
    char* ws = (char*)workspace;
    if (!kept && narrow_backward(c, dy)) return backward_narrow(c, dy, dx, dW, db, ws, st);
    const void* du = dy;
    float* sums = (float*)(ws + p.bytes - up16((int64_t)p.kept_shares * cols * 4));
    if (p.du_bytes && kept) {
        KernelTimer t(KS_GELU, st);
        if (f32) launch_kept_grad<float>(kept, dy, c.n, c.N, c.F, (c.N + p.kept_shares - 1) / p.kept_shares, p.kept_shares, c.act, ws, want_b ? sums : nullptr, st);
        else launch_kept_grad<b16>(kept, dy, c.n, c.N, c.F, (c.N + p.kept_shares - 1) / p.kept_shares, p.kept_shares, c.act, ws, want_b ? sums : nullptr, st);
        TGT_HIP_CHECK(hipGetLastError());
        du = ws;
    } else if (p.du_bytes) {
        Args a = forward_args(c);
        a.dy = dy;
        a.out[0] = ws;
        a.out[1] = c.n == 2 ? ws + c.F * size : nullptr;
        a.out_ld = cols;
        KernelTimer t(KS_LINEAR_FWD, st);
        rc = f32 ? product_forward<float, float>(a, true, Room{}, st) : product_forward<b16, b16>(a, true, Room{}, st);
        if (rc != TGT_OK) return rc;
        du = ws;
    }
    if (dx) {
        Args a{};
        a.P[0] = c.W[0]; a.P[1] = c.n == 2 ? c.W[1] : nullptr;
        a.Q = du;
        a.p_ld = c.K; a.q_ld = cols;
        a.p_count = c.K; a.q_count = c.N;
        a.K = a.K_each = cols; a.K_first = c.F;
        a.out[0] = dx;
        a.out_ld = c.K;
        KernelTimer t(KS_LINEAR_DX, st);
        const Room room{ws + p.du_bytes, p.between};
        rc = f32 ? product_input_grad<float>(a, room, st) : product_input_grad<b16>(a, room, st);
        if (rc != TGT_OK) return rc;
    }
    char* after = ws + p.du_bytes;
    if (want_w) {
        Args a{};
        a.P[0] = c.x;
        a.Q = du;
        a.p_ld = c.K; a.q_ld = cols;
        a.p_count = c.K; a.q_count = cols;
        a.K = a.K_first = c.N;
        a.out[0] = dW[0]; a.out[1] = c.n == 2 ? dW[1] : nullptr;
        a.q_first = c.F;
        a.out_ld = c.K;
        a.partial = (float*)after;
        int splits = 1;
        KernelTimer t(KS_LINEAR_DW, st);
        rc = f32 ? product_weight_grad<float>(a, splits, st) : product_weight_grad<b16>(a, splits, st);
        if (rc != TGT_OK) return rc;
        if (splits >= 16) {      // few elements, many splits: 16 slices of the splits side by side
            tgt_reduce_desc r{};
            r.partial = a.partial; r.workers = splits; r.n = (int)(cols * c.K); r.n_out = c.n;
            r.out[0] = dW[0];
            if (c.n == 2) { r.out[1] = dW[1]; r.begin[1] = c.F * c.K; }
            rc = reduce_partials(&r, 1, c.dtype, st);
            if (rc != TGT_OK) return rc;
        } else if (splits > 1) {
            const int64_t n = cols * c.K, first = (int64_t)c.F * c.K;
            const dim3 grid((unsigned)((n + 1023) / 1024));
            if (f32) hipLaunchKernelGGL((k_add_splits<float>), grid, dim3(256), 0, st, a.partial, splits, n, first, (float*)dW[0], (float*)a.out[1]);
            else hipLaunchKernelGGL((k_add_splits<b16>), grid, dim3(256), 0, st, a.partial, splits, n, first, (b16*)dW[0], (b16*)a.out[1]);
            TGT_HIP_CHECK(hipGetLastError());
        }
    }
    if (want_b) {
        if (!(p.du_bytes && kept)) {
            const dim3 grid((unsigned)((cols + 63) / 64), (unsigned)p.shares);
            if (f32) hipLaunchKernelGGL((k_column_sums<float>), grid, dim3(256), 0, st, (const float*)du, c.N, cols, p.rows_each, sums);
            else hipLaunchKernelGGL((k_column_sums<b16>), grid, dim3(256), 0, st, (const b16*)du, c.N, cols, p.rows_each, sums);
            TGT_HIP_CHECK(hipGetLastError());
        }
        tgt_reduce_desc r{};
        r.partial = sums; r.workers = p.du_bytes && kept ? p.kept_shares : p.shares; r.n = (int)cols; r.n_out = c.n;
        r.out[0] = db[0]; r.begin[0] = 0;
        if (c.n == 2) { r.out[1] = db[1]; r.begin[1] = c.F; }
        return reduce_partials(&r, 1, c.dtype, st);
    }
    return TGT_OK;
}

int64_t kept_room(int n, int64_t N, int F, int dtype) { return N * n * (dtype == TGT_DTYPE_F32 ? kept_width<float>(F) * 4 : kept_width<b16>(F) * 2); }
int64_t kept_bytes_of(int n, int64_t N, int K, int F, int dtype, int act) {
    if (N < 0 || K < 1 || F < 1 || (dtype != TGT_DTYPE_F32 && dtype != TGT_DTYPE_BF16)) return -1;
    const Call c{"", nullptr, {nullptr, nullptr}, {nullptr, nullptr}, n, N, K, F, dtype, act};
    return keeps(c) ? kept_room(n, N, F, dtype) : 0;
}
int64_t fwd_bytes_of(int n, int64_t N, int K, int F, int dtype, bool bits8) {
    if (N < 0 || K < 1 || F < 1 || (dtype != TGT_DTYPE_F32 && dtype != TGT_DTYPE_BF16)) return -1;
    if (few_rows(N, F)) return 0;
    return bits8 ? room_of<e4m3>(F, N, K, n) : dtype == TGT_DTYPE_F32 ? room_of<float>(F, N, K, n) : room_of<b16>(F, N, K, n);
}
int64_t workspace_bytes_of(int n, int64_t N, int K, int F, int dtype, int act) {
    if (N < 0 || K < 1 || F < 1 || (dtype != TGT_DTYPE_F32 && dtype != TGT_DTYPE_BF16)) return -1;
    if (N == 0) return 0;
    // (what decides which way a call goes is in part where its tensors lie: room for either)
    const Call c{"", nullptr, {nullptr, nullptr}, {nullptr, nullptr}, n, N, K, F, dtype, act};
    const int64_t general = plan_of(n, N, K, F, dtype, act).bytes;
    return narrow(c) ? std::max(general, narrow_bytes(n, N, K, F, dtype, act)) : general;
}

}  // namespace
#endif
}  // namespace tgt

#if TGT_GATED_PART == 0
extern "C" {

int tgt_gated_linear_fwd(const void* d_x, const void* d_Wg, const void* d_Wu, const void* d_bg, const void* d_bu, int64_t N, int in_features, int out_features,
                         int dtype, int act, void* d_h, void* d_kept, void* d_workspace, int64_t workspace_bytes, void* stream) {
    const tgt::Call c{"tgt_gated_linear_fwd", d_x, {d_Wg, d_Wu}, {d_bg, d_bu}, 2, N, in_features, out_features, dtype, act};
    return tgt::forward(c, nullptr, d_h, d_kept, {d_workspace, workspace_bytes}, (hipStream_t)stream);
}
int64_t tgt_gated_linear_fwd_workspace_bytes(int64_t N, int in_features, int out_features, int dtype) {
    return tgt::fwd_bytes_of(2, N, in_features, out_features, dtype, false);
}
int64_t tgt_gated_linear_8bit_workspace_bytes(int64_t N, int in_features, int out_features) {
    return tgt::fwd_bytes_of(2, N, in_features, out_features, TGT_DTYPE_F32, true);
}
int64_t tgt_gated_linear_kept_bytes(int64_t N, int in_features, int out_features, int dtype, int act) {
    return tgt::kept_bytes_of(2, N, in_features, out_features, dtype, act);
}
int tgt_gated_linear_8bit_fwd(const void* d_x, const float* d_x_scales, const void* d_Wg, const float* d_Wg_scales, const void* d_Wu, const float* d_Wu_scales,
                              const void* d_bg, const void* d_bu, int64_t N, int in_features, int out_features, int dtype, int act, void* d_h, void* d_workspace,
                              int64_t workspace_bytes, void* stream) {
    const tgt::Call c{"tgt_gated_linear_8bit_fwd", d_x, {d_Wg, d_Wu}, {d_bg, d_bu}, 2, N, in_features, out_features, dtype, act};
    return tgt::forward_8bit(c, d_x_scales, d_Wg_scales, d_Wu_scales, nullptr, d_h, {d_workspace, workspace_bytes}, (hipStream_t)stream);
}
int64_t tgt_gated_linear_bwd_workspace_bytes(int64_t N, int in_features, int out_features, int dtype) {
    return tgt::workspace_bytes_of(2, N, in_features, out_features, dtype, TGT_ACT_SILU);
}
int tgt_gated_linear_bwd(const void* d_x, const void* d_Wg, const void* d_Wu, const void* d_bg, const void* d_bu, const void* d_dh, int64_t N, int in_features,
                         int out_features, int dtype, int act, const void* d_kept, void* d_dx, void* const* d_dW, void* const* d_db, void* d_workspace,
                         int64_t workspace_bytes, void* stream) {
    const tgt::Call c{"tgt_gated_linear_bwd", d_x, {d_Wg, d_Wu}, {d_bg, d_bu}, 2, N, in_features, out_features, dtype, act};
    return tgt::backward(c, d_kept, d_dh, d_dx, d_dW, d_db, d_workspace, workspace_bytes, (hipStream_t)stream);
}

int tgt_linear_epilogue_fwd(const void* d_x, const void* d_W, const void* d_b, const void* d_residual, int64_t N, int in_features, int out_features, int dtype,
                            int act, void* d_y, void* d_kept, void* d_workspace, int64_t workspace_bytes, void* stream) {
    const tgt::Call c{"tgt_linear_epilogue_fwd", d_x, {d_W, nullptr}, {d_b, nullptr}, 1, N, in_features, out_features, dtype, act};
    return tgt::forward(c, d_residual, d_y, d_kept, {d_workspace, workspace_bytes}, (hipStream_t)stream);
}
int64_t tgt_linear_epilogue_fwd_workspace_bytes(int64_t N, int in_features, int out_features, int dtype) {
    return tgt::fwd_bytes_of(1, N, in_features, out_features, dtype, false);
}
int64_t tgt_linear_epilogue_8bit_workspace_bytes(int64_t N, int in_features, int out_features) {
    return tgt::fwd_bytes_of(1, N, in_features, out_features, TGT_DTYPE_F32, true);
}
int64_t tgt_linear_epilogue_kept_bytes(int64_t N, int in_features, int out_features, int dtype, int act) {
    return tgt::kept_bytes_of(1, N, in_features, out_features, dtype, act);
}
int tgt_linear_epilogue_8bit_fwd(const void* d_x, const float* d_x_scales, const void* d_W, const float* d_W_scales, const void* d_b, const void* d_residual,
                                 int64_t N, int in_features, int out_features, int dtype, int act, void* d_y, void* d_workspace, int64_t workspace_bytes,
                                 void* stream) {
    const tgt::Call c{"tgt_linear_epilogue_8bit_fwd", d_x, {d_W, nullptr}, {d_b, nullptr}, 1, N, in_features, out_features, dtype, act};
    return tgt::forward_8bit(c, d_x_scales, d_W_scales, nullptr, d_residual, d_y, {d_workspace, workspace_bytes}, (hipStream_t)stream);
}
int64_t tgt_linear_epilogue_bwd_workspace_bytes(int64_t N, int in_features, int out_features, int dtype, int act) {
    return tgt::workspace_bytes_of(1, N, in_features, out_features, dtype, act);
}
int tgt_linear_epilogue_bwd(const void* d_x, const void* d_W, const void* d_b, const void* d_dy, int64_t N, int in_features, int out_features, int dtype, int act,
                            const void* d_kept, void* d_dx, void* d_dW, void* d_db, void* d_workspace, int64_t workspace_bytes, void* stream) {
    const tgt::Call c{"tgt_linear_epilogue_bwd", d_x, {d_W, nullptr}, {d_b, nullptr}, 1, N, in_features, out_features, dtype, act};
    void *dW[2] = {d_dW, nullptr}, *db[2] = {d_db, nullptr};
    return tgt::backward(c, d_kept, d_dy, d_dx, dW, db, d_workspace, workspace_bytes, (hipStream_t)stream);
}

}  // extern "C"
#endif
