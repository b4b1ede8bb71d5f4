// Gated projections and linears with an epilogue, forward and the first kernel of the backward, where the widths are small and the nodes many:
// the arithmetic and the layouts of linear_tiles.hip with both weights' sums of an output piece in the registers of one wave.
//
//   h = act(g) * u, y = act(g) + residual;   dg = dh u act'(g), du = dh act(g), with g = x W0^T + b0, u = x W1^T + b1
//
// A wave takes 32 node rows; their features become matrix operands in its registers (float32 as three exact bf16 planes, six products, the five
// small ones in a sum of their own), 64 x 64 pieces of the weights go through LDS, shared by the workgroup's four waves, and 64 columns of g and of u
// accumulate side by side.  What else an output needs (the gradient of h, a residual) is asked for before the products.  x of up to 64
// features stays in registers for all columns.  Bound by vector instructions (activations, cutting into planes: about half the time) and the traffic of
// x, h and the gradients.  64000 x 64 -> 128 float32, gelu: forward 26 us (49 MB), gradients 31 us (131 MB); through tiles of 128 x 128 35 and 51 us, and
// 40 and 88 with a gradient's piece in registers of its own (256 are not enough) and 1 KB of LDS more than two workgroups on a CU have.
#include "gated_tiles.h"
#include "activations.h"
#include "linear_pieces.h"
#include <algorithm>

namespace tgt {
namespace {

constexpr int kThreads = 256, kWaves = 4;
template <typename T> constexpr int narrow_lds() { return 2 * kFragVecs<Num<T>::P> * 16 + kWaves * RowShape<T>::kVecs * 16; }      // (float32: 80 KB, two workgroups per CU)

// As fetch_cols and put_cols; WHOLE false: rows that need not be multiples of 16 bytes, element by element
template <typename T, bool WHOLE> __device__ __forceinline__ void fetch_any(Raw<T>& raw, const T* __restrict__ src, int ld, int c0, const Rows& rows, int lane) {
    if (WHOLE) { fetch_cols(raw, src, ld, c0, rows, lane); return; }
    constexpr int PP = RowShape<T>::kPieces, PER = RowShape<T>::kPer, VE = 16 / (int)sizeof(T);
    const int last = rows.left > 0 ? rows.left - 1 : 0, r0 = lane / PP, col = c0 + (lane % PP) * VE;
#pragma unroll
    for (int i = 0; i < RowShape<T>::kAcc; ++i) {
        const int r = r0 + i * PER;
        const T* p = src + (rows.first + (r < last ? r : last)) * ld;
        union { T e[VE]; vec16 v; } u;
        u.v = vec16{0u, 0u, 0u, 0u};
#pragma unroll
        for (int e = 0; e < VE; ++e)
            if (col + e < ld) u.e[e] = p[col + e];
        raw.v[i] = u.v;
    }
}
// The wave's image of its rows in LDS from and to memory (the register side is by node: node_base)
template <typename T> __device__ __forceinline__ void image_of(vec16* stage, const Raw<T>& raw, int lane) {
    wave_sync();
    const int rb = row_base<T>(lane);
#pragma unroll
    for (int i = 0; i < RowShape<T>::kAcc; ++i) stage[row_slot<T>(rb, i)] = raw.v[i];
    wave_sync();
}
template <typename T, bool WHOLE> __device__ __forceinline__ void put_image(T* __restrict__ dst, int ld, int c0, const vec16* stage, const Rows& rows, int lane) {
    constexpr int PP = RowShape<T>::kPieces, PER = RowShape<T>::kPer, VE = 16 / (int)sizeof(T);
    wave_sync();
    const int rb = row_base<T>(lane), r0 = lane / PP, col = c0 + (lane % PP) * VE;
    T* p = dst + (rows.first + r0) * ld + col;
    if constexpr (WHOLE) {
        vec16 v[RowShape<T>::kAcc];
#pragma unroll
        for (int i = 0; i < RowShape<T>::kAcc; ++i) v[i] = stage[row_slot<T>(rb, i)];
        if (col >= ld) return;
#pragma unroll
        for (int i = 0; i < RowShape<T>::kAcc; ++i)
            if (r0 + i * PER < rows.left) *reinterpret_cast<vec16*>(p + (int64_t)(i * PER) * ld) = v[i];
    } else {
#pragma unroll
        for (int i = 0; i < RowShape<T>::kAcc; ++i) {
            union { T e[VE]; vec16 v; } u;
            u.v = stage[row_slot<T>(rb, i)];
#pragma unroll
            for (int e = 0; e < VE; ++e)
                if (r0 + i * PER < rows.left && col + e < ld) p[(int64_t)(i * PER) * ld + e] = u.e[e];
        }
    }
}

// Sums that an infinity went through (see holds_nan): once more in plain multiply-adds, by way of the wave's place in LDS (indexed registers
// would be scratch memory for every wave)
template <typename T> __device__ __forceinline__ void mend(Tile& t, const NarrowArgs& a, int w, int c0, vec16* stage, const Rows& rows, int lane) {
    if constexpr (Num<T>::P == 3) {
        if (!holds_nan([&](int i) { return t.get(i); }, 32)) return;
        const int nb = node_base<T>(lane), n = lane & 31;
        wave_sync();
#pragma unroll
        for (int i = 0; i < 8; ++i) stage[nb ^ i] = vec16{__float_as_uint(t.get(4 * i)), __float_as_uint(t.get(4 * i + 1)), __float_as_uint(t.get(4 * i + 2)), __float_as_uint(t.get(4 * i + 3))};
        const float* x = reinterpret_cast<const float*>(a.x) + (rows.first + (n < rows.left ? n : 0)) * a.K;
#pragma unroll 1
        for (int i = 0; i < 32; ++i) {
            float* v = reinterpret_cast<float*>(stage + (nb ^ (i >> 2))) + (i & 3);
            const int c = c0 + 32 * (lane >> 5) + i;
            if (n < rows.left && c < a.F && !(fabsf(*v) < __builtin_inff())) {
                const float* W = reinterpret_cast<const float*>(a.W[w]) + (int64_t)c * a.K;
                float s = a.bias[w] ? reinterpret_cast<const float*>(a.bias[w])[c] : 0.f;
                for (int k = 0; k < a.K; ++k) s = fmaf(x[k], W[k], s);
                *v = s;
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const vec16 v = stage[nb ^ i];
#pragma unroll
            for (int e = 0; e < 4; ++e) t.set(4 * i + e, __uint_as_float(v[e]));
        }
        wave_sync();
    }
}

// The sums of a piece to what is written, one 16-byte piece of the lane's row at a time in the wave's image of the rows, which holds the residual or
// the result's gradient (`more`) and then the result or dg.  du stays in acc[1].
template <typename T, bool TWO, bool GRAD, int ACT> __device__ __forceinline__ void combine(Tile (&acc)[TWO ? 2 : 1], vec16* stage, bool more, int lane) {
    constexpr bool EXACT = sizeof(T) == 4;
    constexpr int VE = 16 / (int)sizeof(T);
    const int nb = node_base<T>(lane);
#pragma unroll
    for (int i = 0; i < 32 / VE; ++i) {
        float in[VE], o[VE];
        if (GRAD || (!TWO && more)) unpack16(stage[nb ^ i], in, (const T*)nullptr);
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            const int at = i * VE + e;
            const float g = acc[0].get(at);
            if constexpr (GRAD && TWO) {
                float a, s;
                act_and_slope<EXACT, ACT>(g, a, s);
                o[e] = in[e] * acc[1].get(at) * s;
                acc[1].set(at, in[e] * a);
            } else if constexpr (GRAD) o[e] = slope_of<EXACT, ACT>(g, in[e]);
            else if constexpr (TWO) o[e] = act_of<EXACT, ACT>(g) * acc[1].get(at);
            else o[e] = more ? act_of<EXACT, ACT>(g) + in[e] : act_of<EXACT, ACT>(g);
        }
        stage[nb ^ i] = pack16(o, (const T*)nullptr);
        fence_schedule();      // (side by side, thirty-two of them have no registers)
    }
}

// blockIdx.x: 128 rows; blockIdx.y: `per` of the 64-column pieces.  RES: 64-feature pieces of x that stay in registers (0: none)
template <typename T, bool TWO, bool GRAD, int RES, bool WHOLE>
__global__ __launch_bounds__(kThreads, 2) void k_gated_tiles(const NarrowArgs a, const int per) {
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int P = Num<T>::P, FV = kFragVecs<P>, NW = TWO ? 2 : 1;
    constexpr bool READS = GRAD || !TWO, EARLY = READS && !(P == 3 && (TWO || RES == 2));      // (float32: no registers for it beside two sums or two pieces of x)
    vec16* w = reinterpret_cast<vec16*>(smem);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    vec16* stage = w + 2 * FV + wave * RowShape<T>::kVecs;
    const int nk = (a.K + 63) / 64, nc = ((GRAD ? a.out_ld : a.F) + 63) / 64;
    const int first = blockIdx.y * per, end = first + per < nc ? first + per : nc;
    const Rows rows((int64_t)blockIdx.x * kWaves + wave, a.N);
    const T* const x = reinterpret_cast<const T*>(a.x);
    const T* const more = reinterpret_cast<const T*>(a.more);
    if constexpr (GRAD && !TWO) {
        if (a.padded) {      // (a launch of its own costs more than the copy)
            constexpr int VE = 16 / (int)sizeof(T);
            const int all = (int)((int64_t)a.out_ld * a.K / VE), have = (int)((int64_t)a.F * a.K / VE), by = (int)(gridDim.x * gridDim.y) * kThreads;
            for (int i = (int)(blockIdx.y * gridDim.x + blockIdx.x) * kThreads + (int)threadIdx.x; i < all; i += by)
                reinterpret_cast<vec16*>(a.padded)[i] = i < have ? reinterpret_cast<const vec16*>(a.W[0])[i] : vec16{0u, 0u, 0u, 0u};
        }
    }
    Frags<P> f[RES ? RES : 1];
    Raw<T> raw;
    const auto operands = [&](Frags<P>& to) {
        Tile t;
        settle<T, false>(t, raw, stage, rows, lane);
        make_frags(to, t);
    };
    fetch_cols(raw, x, a.K, 0, rows, lane);
    Piece<T> next;
    const auto ask = [&](int t, int o, int k) { fetch_piece<T, false>(next, reinterpret_cast<const T*>(a.W[o]), a.K, t * 64, a.F, k * 64, a.K); };
    if constexpr (RES > 0) {
#pragma unroll
        for (int k = 0; k < RES; ++k) {
            operands(f[k]);
            if (k + 1 < RES) fetch_cols(raw, x, a.K, 64 * (k + 1), rows, lane);
        }
    }
    ask(first, 0, 0);
    const auto bias_of = [&](int t, int o) {
        const int c = t * 64 + lane;
        return a.bias[o] && c < a.F ? as_float(reinterpret_cast<const T*>(a.bias[o])[c]) : 0.f;
    };
    float bias[NW];
#pragma unroll
    for (int o = 0; o < NW; ++o) bias[o] = bias_of(first, o);
    int turn = 0;
    for (int t = first; t < end; ++t) {
        const int c0 = t * 64;
        Raw<T> raw_in;
        if (EARLY && more) fetch_any<T, WHOLE>(raw_in, more, a.F, c0, rows, lane);
        Tile acc[NW];
#pragma unroll
        for (int o = 0; o < NW; ++o) {
            // the piece's biases to all lanes by way of the wave's place in LDS
            wave_sync();
            reinterpret_cast<float*>(stage)[lane] = bias[o];
            wave_sync();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const vec16 v = stage[8 * (lane >> 5) + i];
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[o].set(4 * i + e, __uint_as_float(v[e]));
            }
            if (t + 1 < end) bias[o] = bias_of(t + 1, o);
            for (int k = 0; k < nk; ++k, turn ^= 1) {
                vec16* const mine = w + turn * FV;      // last read in the step before the one before: every wave has passed the barrier since
                put_piece<T, P>(mine, next, c0, a.F, k * 64, a.K);
                if (k + 1 < nk) ask(t, o, k + 1);
                else if (o + 1 < NW) ask(t, o + 1, 0);
                else if (t + 1 < end) ask(t + 1, 0, 0);
                if constexpr (RES == 0) {
                    operands(f[0]);
                    if (k + 1 < nk || o + 1 < NW || t + 1 < end) fetch_cols(raw, x, a.K, k + 1 < nk ? 64 * (k + 1) : 0, rows, lane);
                }
                __syncthreads();
                if (RES == 2 && k == 1) gemm_apart<P>(acc[o], f[RES == 2 ? 1 : 0], mine, lane);
                else gemm_apart<P>(acc[o], f[0], mine, lane);
            }
            mend<T>(acc[o], a, o, c0, stage, rows, lane);
        }
        if (READS && !EARLY && more) fetch_any<T, WHOLE>(raw_in, more, a.F, c0, rows, lane);
        if (READS && more) image_of<T>(stage, raw_in, lane);
        else wave_sync();
        switch (a.act) {
            case TGT_ACT_SILU: combine<T, TWO, GRAD, TGT_ACT_SILU>(acc, stage, more, lane); break;
            case TGT_ACT_GELU: combine<T, TWO, GRAD, TGT_ACT_GELU>(acc, stage, more, lane); break;
            case TGT_ACT_RELU: combine<T, TWO, GRAD, TGT_ACT_RELU>(acc, stage, more, lane); break;
            default: combine<T, TWO, GRAD, TGT_ACT_NONE>(acc, stage, more, lane); break;
        }
        put_image<T, WHOLE || GRAD>(reinterpret_cast<T*>(a.out[0]), a.out_ld, c0, stage, rows, lane);
        if constexpr (TWO && GRAD) put_cols(reinterpret_cast<T*>(a.out[1]), a.out_ld, c0, acc[NW - 1], stage, rows, lane);
    }
}

template <typename T, bool TWO, bool GRAD, int RES, bool WHOLE> int launch(const NarrowArgs& a, hipStream_t st) {
    static std::atomic<uint64_t> done{0};
    constexpr int lds = narrow_lds<T>();
    if (int rc = allow_lds(reinterpret_cast<const void*>(&k_gated_tiles<T, TWO, GRAD, RES, WHOLE>), lds, done)) return rc;
    // two workgroups per CU: below that the columns are shared out
    const int64_t panels = (a.N + 32 * kWaves - 1) / (32 * kWaves);
    const int nc = ((GRAD ? a.out_ld : a.F) + 63) / 64, splits = (int)std::min<int64_t>(nc, std::max<int64_t>(1, 512 / panels)), per = (nc + splits - 1) / splits;
    hipLaunchKernelGGL((k_gated_tiles<T, TWO, GRAD, RES, WHOLE>), dim3((unsigned)panels, (unsigned)((nc + per - 1) / per)), dim3(kThreads), lds, st, a, per);
    TGT_HIP_CHECK(hipGetLastError());
    return TGT_OK;
}
template <typename T, bool TWO, bool GRAD> int run(const NarrowArgs& a, hipStream_t st) {
    // (the gradients' rows are the caller's own, whole ones; what they are made of and results are a user's)
    const bool whole = a.F % (16 / (int)sizeof(T)) == 0 && ((uintptr_t)a.more & 15) == 0 && (GRAD || ((uintptr_t)a.out[0] & 15) == 0);
    if (a.K <= 64) return whole ? launch<T, TWO, GRAD, 1, true>(a, st) : launch<T, TWO, GRAD, 1, false>(a, st);
    // (two pieces of x take 96 registers in float32, which the gradients do not leave)
    if constexpr (!GRAD)
        if (a.K <= 128) return whole ? launch<T, TWO, GRAD, 2, true>(a, st) : launch<T, TWO, GRAD, 2, false>(a, st);
    return whole ? launch<T, TWO, GRAD, 0, true>(a, st) : launch<T, TWO, GRAD, 0, false>(a, st);
}
template <typename T> int pick(const NarrowArgs& a, bool grad, hipStream_t st) {
    if (a.W[1]) return grad ? run<T, true, true>(a, st) : run<T, true, false>(a, st);
    return grad ? run<T, false, true>(a, st) : run<T, false, false>(a, st);
}

}  // namespace

int gated_tiles(const NarrowArgs& a, bool grad, int dtype, hipStream_t st) {
    return dtype == TGT_DTYPE_F32 ? pick<float>(a, grad, st) : pick<nbf16>(a, grad, st);
}

}  // namespace tgt
