// Rows of a matrix of any width and 64 x 64 pieces of a weight on their way to matrix operands (layouts of node_tile.h), for the linears of
// linear_tiles.hip and the gated projections of gated_tiles.hip.
#pragma once
#include "node_tile.h"

namespace tgt {
namespace {

// 16 bytes of row r's columns k0 + ... of an array with ld columns (16-byte pieces; K of them count)
template <typename T> __device__ __forceinline__ void fetch_cols(Raw<T>& raw, const T* __restrict__ src, int ld, int k0, const Rows& rows, int lane) {
    constexpr int PP = RowShape<T>::kPieces, PER = RowShape<T>::kPer, VE = 16 / (int)sizeof(T);
    const int last = rows.left > 0 ? rows.left - 1 : 0, r0 = lane / PP, col = k0 + (lane % PP) * VE;
    const T* p = src + rows.first * ld + (col < ld ? col : 0);
#pragma unroll
    for (int i = 0; i < RowShape<T>::kAcc; ++i) {
        const int r = r0 + i * PER;
        raw.v[i] = *reinterpret_cast<const vec16*>(p + (int64_t)(r < last ? r : last) * ld);
    }
    if (k0 + 64 > ld && col >= ld) {      // (the weights are zero there, the row's neighbour may be anything)
#pragma unroll
        for (int i = 0; i < RowShape<T>::kAcc; ++i) raw.v[i] = vec16{0u, 0u, 0u, 0u};
    }
}
template <typename T> __device__ __forceinline__ void put_cols(T* __restrict__ dst, int ld, int c0, const Tile& t, vec16* stage, const Rows& rows, int lane) {
    constexpr int PP = RowShape<T>::kPieces, PER = RowShape<T>::kPer, VE = 16 / (int)sizeof(T);
    wave_sync();
    const int nb = node_base<T>(lane);
#pragma unroll
    for (int i = 0; i < PP / 2; ++i) {
        float f[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) f[e] = t.get(i * VE + e);
        stage[nb ^ i] = pack16(f, (const T*)nullptr);
    }
    wave_sync();
    const int rb = row_base<T>(lane), r0 = lane / PP, col = c0 + (lane % PP) * VE;
    vec16 v[RowShape<T>::kAcc];
#pragma unroll
    for (int i = 0; i < RowShape<T>::kAcc; ++i) v[i] = stage[row_slot<T>(rb, i)];
    if (col >= ld) return;
    T* p = dst + rows.first * ld + col;
#pragma unroll
    for (int i = 0; i < RowShape<T>::kAcc; ++i)
        if (r0 + i * PER < rows.left) *reinterpret_cast<vec16*>(p + (int64_t)(r0 + i * PER) * ld) = v[i];
}

// A thread's share of a 64 x 64 piece of the weight on its way to LDS: two operand vectors (outputs o0 .., contraction k0 ..)
template <typename T> struct Piece { T v[2][8]; };
template <typename T, bool DX> __device__ __forceinline__ void fetch_piece(Piece<T>& w, const T* __restrict__ W, int ld, int o0, int outs, int k0, int len) {
    const int lane = forgotten(threadIdx.x & 63), r = lane & 31;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int sm = (threadIdx.x >> 6) + 4 * j, s = sm >> 1, m = sm & 1;
        int o = o0 + 32 * ((r >> 2) & 1) + 16 * m + 4 * (r >> 3) + (r & 3), k = k0 + 32 * (lane >> 5) + 8 * s;
        o = o < outs ? o : outs - 1;
        if (DX) {      // eight rows of W at one column
            if (k0 + 64 <= len) {      // (one vector offset, the rows as scalar bases)
                const uint32_t at = k * ld + o;
#pragma unroll
                for (int i = 0; i < 8; ++i) w.v[j][i] = (W + i * ld)[at];
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) w.v[j][i] = W[(uint32_t)((k + i < len ? k + i : len - 1) * ld + o)];
            }
        } else {       // eight columns of one row, in 16-byte pieces that end with the row
            constexpr int VE = 16 / (int)sizeof(T);
#pragma unroll
            for (int q = 0; q < 8 / VE; ++q) {
                const int c = k + q * VE;
                *reinterpret_cast<vec16*>(&w.v[j][q * VE]) = *reinterpret_cast<const vec16*>(W + (uint32_t)(o * ld + (c < len ? c : len - VE)));
            }
        }
    }
}
template <typename T, int P> __device__ __forceinline__ void put_piece(vec16* dst, const Piece<T>& w, int o0, int outs, int k0, int len) {
    const int lane = forgotten(threadIdx.x & 63), r = lane & 31;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int sm = (threadIdx.x >> 6) + 4 * j, s = sm >> 1, m = sm & 1;
        const int o = o0 + 32 * ((r >> 2) & 1) + 16 * m + 4 * (r >> 3) + (r & 3), k = k0 + 32 * (lane >> 5) + 8 * s;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = o < outs && k + i < len ? as_float(w.v[j][i]) : 0.f;
        bf16x8_t p[P];
        to_planes(v, p);
#pragma unroll
        for (int q = 0; q < P; ++q) dst[(sm * P + q) * 64 + lane] = __builtin_bit_cast(vec16, p[q]);
    }
}

}  // namespace
}  // namespace tgt
