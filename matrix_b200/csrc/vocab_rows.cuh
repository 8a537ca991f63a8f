// Rows of logits: what the vocabulary operators (distill.cu, sampling.cu) share.
//
// A batch of logits is rows of V contiguous elements; row r lies at
// (r / rows_inner) * stride_outer + (r % rows_inner) * stride_inner, so a
// shifted or padded view (logits[:, :-1], logits[..., :V]) is read in place.
// A row may start on any element.  It is read in 16-byte words counted from the
// boundary at or before its first element: word g holds the elements
// [g * VEC - shift, (g + 1) * VEC - shift), of which the first and the last word
// may hold some outside [0, V); those two are read element by element and
// nothing outside the row is touched.
#pragma once

#include "dwa_common.cuh"

namespace dwa {

constexpr float kLog2e = 1.4426950408889634f;

template <class T> constexpr int kRowVec = 16 / static_cast<int>(sizeof(T));

__device__ __forceinline__ int64_t row_offset(const DwaLogitsDims& d, int64_t r) {
    return (r / d.rows_inner) * d.stride_outer + (r % d.rows_inner) * d.stride_inner;
}

template <class T>
__device__ __forceinline__ void unpack(uint4 w, float* v) {
    if constexpr (sizeof(T) == 2) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(u[i] << 16);
            v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        }
    } else {
        v[0] = __uint_as_float(w.x);
        v[1] = __uint_as_float(w.y);
        v[2] = __uint_as_float(w.z);
        v[3] = __uint_as_float(w.w);
    }
}

template <class T>
__device__ __forceinline__ uint4 pack(const float* v) {
    if constexpr (sizeof(T) == 2) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            u[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        return make_uint4(u[0], u[1], u[2], u[3]);
    } else {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
}

// The words of one row.
template <class T>
struct RowWords {
    const T* row;
    int V, shift, words, full_lo, full_hi;   // words [full_lo, full_hi) lie whole inside the row

    __device__ __forceinline__ RowWords(const T* p, int V_) : row(p), V(V_) {
        constexpr int VEC = kRowVec<T>;
        shift = static_cast<int>(reinterpret_cast<uintptr_t>(p) % 16) / static_cast<int>(sizeof(T));
        words = (V + shift + VEC - 1) / VEC;
        full_lo = shift > 0 ? 1 : 0;
        full_hi = (V + shift) / VEC;
    }
    __device__ __forceinline__ int first(int g) const { return g * kRowVec<T> - shift; }
    __device__ __forceinline__ uint4 word(int g) const { return *reinterpret_cast<const uint4*>(row + first(g)); }
    // a first or last word: -inf outside the row
    __device__ __forceinline__ void edge(int g, float* v) const {
#pragma unroll
        for (int i = 0; i < kRowVec<T>; ++i) {
            const int j = first(g) + i;
            v[i] = (j >= 0 && j < V) ? Elem<T>::to_f(row[j]) : -INFINITY;
        }
    }

    // f(v, j0) for every word of [lo, hi) in this thread's share (threads tid of
    // n): the word's VEC values and its first index.  U words are in flight.
    template <int U, class F>
    __device__ __forceinline__ void each(int lo, int hi, int tid, int n, F f) const {
        constexpr int VEC = kRowVec<T>;
        const int a = lo > full_lo ? lo : full_lo, b = hi < full_hi ? hi : full_hi;
        int g = a + tid;
        for (; g + (U - 1) * n < b; g += U * n) {
            uint4 w[U];
#pragma unroll
            for (int u = 0; u < U; ++u) w[u] = word(g + u * n);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float v[VEC];
                unpack<T>(w[u], v);
                f(v, first(g + u * n));
            }
        }
        for (; g < b; g += n) {
            float v[VEC];
            unpack<T>(word(g), v);
            f(v, first(g));
        }
        if (tid < 2) {   // thread 0 the first word, thread 1 the last, where they are not whole
            const int e = tid == 0 ? 0 : words - 1;
            const bool is_edge = tid == 0 ? full_lo > 0 : (full_hi < words && words - 1 >= full_lo);
            if (is_edge && e >= lo && e < hi) {
                float v[VEC];
                edge(e, v);
                f(v, first(e));
            }
        }
    }
};

// Block-wide reduction in a fixed order; every thread gets the result.  `red`
// holds 33 values; consecutive calls may share it.
template <class V, class Op>
__device__ __forceinline__ V block_reduce(V v, Op op, V identity, V* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    const int w = threadIdx.x >> 5, l = threadIdx.x & 31;
    __syncthreads();
    if (l == 0) red[w] = v;
    __syncthreads();
    if (w == 0) {
        v = l < static_cast<int>(blockDim.x >> 5) ? red[l] : identity;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
        if (l == 0) red[32] = v;
    }
    __syncthreads();
    return red[32];
}

struct MaxOp {
    template <class V> __device__ __forceinline__ V operator()(V a, V b) const { return a > b ? a : b; }
};
struct AddOp {
    template <class V> __device__ __forceinline__ V operator()(V a, V b) const { return a + b; }
};

// The running maximum and sum of exp2((v - m) * c): one pass over the data.
struct MaxSum {
    float m = -INFINITY, s = 0.f;
    __device__ __forceinline__ void raise(float to, float c) {   // m becomes `to` >= m
        if (to > m) {
            s *= exp2f((m - to) * c);   // m = -inf: s is 0 and stays 0
            m = to;
        }
    }
};

int check_logits(const DwaLogitsDims* d, const char* what);   // distill.cu

}  // namespace dwa
