// rope.h — what the rotary operators share (rope.hip: rotation, append; norm_rope.hip: with the heads' norms): a rotation's
// table, rows of values, angles, how a head divides into units.
#pragma once

#include "paged.h"

struct aq_rope {
    aq_ctx *ctx = nullptr;
    uint32_t dim = 0, layout = 0;
    float gain = 1.0f;
    double *freq = nullptr; // dim / 2 turns per position
};

namespace aq {

// N values at p as f32, and back with one rounding; 16 bytes at a time where W.
template <int T, int N, bool W>
__device__ __forceinline__ void load_n(const typename RowType<T>::type *p, float *v) {
    using E = typename RowType<T>::type;
    if constexpr (W) {
        constexpr int C = 16 / (int)sizeof(E);
        typedef E vec __attribute__((ext_vector_type(C)));
#pragma unroll
        for (int i = 0; i < N / C; i++) {
            const vec x = *reinterpret_cast<const vec *>(p + i * C);
#pragma unroll
            for (int j = 0; j < C; j++) v[i * C + j] = (float)x[j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = (float)p[i];
    }
}

template <int T, int N, bool W>
__device__ __forceinline__ void store_n(typename RowType<T>::type *p, const float *v) {
    using E = typename RowType<T>::type;
    if constexpr (W) {
        constexpr int C = 16 / (int)sizeof(E);
        typedef E vec __attribute__((ext_vector_type(C)));
#pragma unroll
        for (int i = 0; i < N / C; i++) {
            vec x;
#pragma unroll
            for (int j = 0; j < C; j++) x[j] = (E)v[i * C + j];
            *reinterpret_cast<vec *>(p + i * C) = x;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) p[i] = (E)v[i];
    }
}

// Sine and cosine of pos * freq turns: the product cut to one turn in 64 bits.
__device__ __forceinline__ void rope_angle(double freq, int32_t pos, float *sn, float *cs) {
    const double t = (double)pos * freq;
    sincospif(2.0f * (float)(t - rint(t)), sn, cs);
}

// How a head divides into units: `vec` values each (half layout: of either half), then the values that pass through.
inline void unit_shape(uint32_t layout, uint32_t dim, uint32_t hd, uint32_t vec, uint32_t *rot, uint32_t *all) {
    *rot = layout == AQ_ROPE_INTERLEAVED ? dim / vec : dim / 2 / vec;
    *all = *rot + (hd - dim) / vec;
}
inline bool wide_fits(uint32_t layout, uint32_t dim, uint32_t hd, uint32_t vec) {
    return hd % vec == 0 && dim % vec == 0 && (layout == AQ_ROPE_INTERLEAVED || (dim / 2) % vec == 0);
}

} // namespace aq
