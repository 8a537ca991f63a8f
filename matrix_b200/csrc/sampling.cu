// The largest logits of a row, and sampling from a row.
//
// Both order the entries of a row by one 64-bit key: the logit (as an ordered
// 32-bit integer, -0 as +0, NaN above everything) over the complement of the
// index, so that larger logits come first, equal ones by index, and no two keys
// are equal.  "The k largest" and "the shortest prefix that holds a mass" are
// then one key each: everything at or above it is kept.
//
// Sampling, for a row z [V] and given numbers e [V] drawn from the exponential
// distribution: w_i = exp((z_i - max z) / T); the k largest stay, of these the
// shortest leading run whose mass before the entry is below top_p times their
// mass, of these the entries with w_i >= min_p; the token is the one with the
// largest w_i / e_i (an exponential race, which draws i with probability
// w_i / sum w), its log-probability log(w_i / sum of the kept w).
//
// Masses that decide a cut are summed as integers in units of 2^-31 of the
// largest weight: sums that no order of additions changes, so a row's token does
// not depend on how its entries are spread over threads.

#include <atomic>

#include "vocab_rows.cuh"

namespace dwa {

extern std::atomic<uint64_t> g_launches_total;

constexpr int kSelThreads = 512;

// A logit as an unsigned integer of the same order.
__device__ __forceinline__ uint32_t ordered(float z) {
    if (z != z) return 0xffffffffu;
    const uint32_t u = __float_as_uint(z + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t entry_key(float z, int j) {
    return static_cast<uint64_t>(ordered(z)) << 32 | (0xffffffffu - static_cast<uint32_t>(j));
}
__device__ __forceinline__ int key_index(uint64_t key) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(key)); }

// An entry's weight.  1 / T in two floats: the rounding of one would move all
// weights far below the largest the same way, and with them a nucleus' edge.
struct Weigh {
    float m, c, c_lo;
    __device__ __forceinline__ Weigh(float m_, float T) : m(m_) {
        const double cd = 1.4426950408889634 / T;
        c = static_cast<float>(cd);
        c_lo = isinf(c) ? 0.f : static_cast<float>(cd - c);
    }
    __device__ __forceinline__ float operator()(float z) const {
        if (z == m) return 1.f;
        const float d = z - m;
        return z == -INFINITY || m == INFINITY ? 0.f : exp2f(fmaf(d, c, d * c_lo));
    }
    // in units of 2^-31
    __device__ __forceinline__ uint32_t fixed(float z) const { return static_cast<uint32_t>((*this)(z) * 2147483648.f + 0.5f); }
};

// The key at which the entries at or above `floor`, taken in descending order,
// reach `target`: in number (MASS = false) or in mass.  Eight bits of the key a
// pass.  hist: 256 values, found: 2 values in shared memory.
template <class T, bool MASS>
__device__ uint64_t cut_key(const RowWords<T>& w, uint64_t floor, uint64_t target, const Weigh& weigh,
                            unsigned long long* hist, unsigned long long* found) {
    const int tid = threadIdx.x, lane = tid & 31;
    uint64_t prefix = 0, mask = 0;
    int index_bytes = 1;
    while (index_bytes < 4 && (w.V - 1) >> (8 * index_bytes)) ++index_bytes;
    for (int b = 7; b >= 0; --b) {
        const int shift = 8 * b;
        if (b < 4 && b >= index_bytes) {   // the complement of an index below 256^b: all ones
            prefix |= uint64_t(0xff) << shift;
            mask |= uint64_t(0xff) << shift;
            continue;
        }
        __syncthreads();
        for (int i = tid; i < 256; i += blockDim.x) hist[i] = 0ull;
        __syncthreads();
        w.template each<2>(0, w.words, tid, blockDim.x, [&](const float* v, int j0) {
#pragma unroll
            for (int i = 0; i < kRowVec<T>; ++i) {
                const uint64_t key = entry_key(v[i], j0 + i);
                if (static_cast<unsigned>(j0 + i) < static_cast<unsigned>(w.V) && key >= floor && (key & mask) == prefix) {
                    const uint32_t digit = static_cast<uint32_t>(key >> shift) & 0xffu;
                    const unsigned peers = __match_any_sync(__activemask(), digit);
                    unsigned long long sum;
                    if (MASS) {
                        const uint32_t x = weigh.fixed(v[i]);
                        sum = (static_cast<unsigned long long>(__reduce_add_sync(peers, x >> 16)) << 16) +
                              __reduce_add_sync(peers, x & 0xffffu);
                    } else {
                        sum = __popc(peers);
                    }
                    if ((peers & ((1u << lane) - 1u)) == 0u) atomicAdd(&hist[digit], sum);
                }
            }
        });
        __syncthreads();
        if (tid < 32) {   // lane l: bins 255 - 8l down to 248 - 8l
            unsigned long long own = 0ull;
#pragma unroll
            for (int i = 0; i < 8; ++i) own += hist[255 - 8 * lane - i];
            unsigned long long incl = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned long long up = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += up;
            }
            unsigned long long acc = incl - own;
            if (acc < target && target <= incl) {
                int d = 255 - 8 * lane;
                while (acc + hist[d] < target) acc += hist[d--];
                found[0] = static_cast<unsigned long long>(d);
                found[1] = acc;
            }
        }
        __syncthreads();
        prefix |= found[0] << shift;
        mask |= uint64_t(0xff) << shift;
        target -= found[1];
    }
    return prefix;
}

// ---------------------------------------------------------------------------
// the largest logits
// ---------------------------------------------------------------------------
struct TopArgs {
    const void* z;
    DwaLogitsDims d;
    int K;
    float c, temperature;
    void* values;
    int32_t* indices;
    float* lse;
};

// A row's maximum and sum of exp((z - max) c); `nan` tells whether one is there.
template <class T>
__device__ MaxSum row_max_sum(const RowWords<T>& w, float c, float* red, bool& nan) {
    MaxSum ms;
    w.template each<4>(0, w.words, threadIdx.x, blockDim.x, [&](const float* v, int) {
        float top = v[0];
#pragma unroll
        for (int i = 1; i < kRowVec<T>; ++i) top = fmaxf(top, v[i]);
        ms.raise(top, c);
#pragma unroll
        for (int i = 0; i < kRowVec<T>; ++i) ms.s += v[i] == -INFINITY ? 0.f : exp2f((v[i] - ms.m) * c);
    });
    const float m = block_reduce(ms.m, MaxOp(), -INFINITY, red);
    float s = ms.m > -INFINITY ? ms.s * exp2f((ms.m - m) * c) : ms.s;
    ms.s = block_reduce(s, AddOp(), 0.f, red);
    ms.m = m;
    nan = ms.s != ms.s;
    if (m == INFINITY) {   // inf - inf above: look for a NaN itself
        int seen = 0;
        w.template each<1>(0, w.words, threadIdx.x, blockDim.x, [&](const float* v, int) {
#pragma unroll
            for (int i = 0; i < kRowVec<T>; ++i) seen |= v[i] != v[i];
        });
        nan = __syncthreads_or(seen);
    }
    return ms;
}

template <class T>
__global__ void __launch_bounds__(kSelThreads) top_logits_kernel(TopArgs a) {
    pdl_enter();
    __shared__ unsigned long long hist[256], found[2], list[DWA_MAX_TOP];
    __shared__ float red[33];
    __shared__ int count;
    const int tid = threadIdx.x, K = a.K;
    const int64_t r = blockIdx.x;
    const RowWords<T> w(static_cast<const T*>(a.z) + row_offset(a.d, r), a.d.V);
    bool nan;
    const MaxSum ms = row_max_sum(w, a.c, red, nan);
    if (tid == 0) {
        count = 0;
        a.lse[r] = nan ? NAN : isinf(ms.m) ? ms.m : ms.m / a.temperature + logf(ms.s);
    }
    const uint64_t cut = cut_key<T, false>(w, 0, K, Weigh(0.f, 1.f), hist, found);
    w.template each<4>(0, w.words, tid, blockDim.x, [&](const float* v, int j0) {
#pragma unroll
        for (int i = 0; i < kRowVec<T>; ++i) {
            const uint64_t key = entry_key(v[i], j0 + i);
            if (static_cast<unsigned>(j0 + i) < static_cast<unsigned>(w.V) && key >= cut) list[atomicAdd(&count, 1)] = key;
        }
    });
    __syncthreads();
    for (int k = tid; k < K; k += blockDim.x) {
        const unsigned long long key = list[k];
        int rank = 0;
        for (int i = 0; i < K; ++i) rank += list[i] > key;
        const int j = key_index(key);
        static_cast<T*>(a.values)[r * K + rank] = w.row[j];
        a.indices[r * K + rank] = j;
    }
}

// ---------------------------------------------------------------------------
// sampling
// ---------------------------------------------------------------------------
struct SampleArgs {
    const void* z;
    DwaLogitsDims d;
    const float* noise;
    int64_t noise_stride;
    DwaSampleParams p;
    int32_t* tokens;
    float* logprobs;
};

template <class T>
__global__ void __launch_bounds__(kSelThreads) sample_kernel(SampleArgs a) {
    pdl_enter();
    __shared__ unsigned long long hist[256], found[2], red64[33];
    __shared__ float red[33];
    const int tid = threadIdx.x, V = a.d.V;
    const int64_t r = blockIdx.x;
    const RowWords<T> w(static_cast<const T*>(a.z) + row_offset(a.d, r), V);
    const float T0 = a.p.temperature_rows ? a.p.temperature_rows[r] : a.p.temperature;
    const int top_k = a.p.top_k_rows ? a.p.top_k_rows[r] : a.p.top_k;
    const float top_p = a.p.top_p_rows ? a.p.top_p_rows[r] : a.p.top_p;
    const float min_p0 = a.p.min_p_rows ? a.p.min_p_rows[r] : a.p.min_p;
    const float min_p = min_p0 > 0.f ? fminf(min_p0, 1.f) : 0.f;
    const bool greedy = !(T0 > 0.f);
    const float c = greedy ? kLog2e : kLog2e / T0;

    bool nan;
    const MaxSum ms = row_max_sum(w, c, red, nan);
    if (nan || ms.m == -INFINITY) {   // nothing to draw from
        if (tid == 0) {
            a.tokens[r] = -1;
            a.logprobs[r] = NAN;
        }
        return;
    }
    const Weigh weigh(ms.m, greedy ? 1.f : T0);
    uint64_t floor = 0;
    if (!greedy && top_k > 0 && top_k < V) floor = cut_key<T, false>(w, 0, top_k, weigh, hist, found);
    if (!greedy && top_p < 1.f) {
        unsigned long long mass = 0ull;
        w.template each<4>(0, w.words, tid, blockDim.x, [&](const float* v, int j0) {
#pragma unroll
            for (int i = 0; i < kRowVec<T>; ++i)
                if (entry_key(v[i], j0 + i) >= floor) mass += weigh.fixed(v[i]);
        });
        mass = block_reduce(mass, AddOp(), 0ull, red64);
        const double want = ceil(static_cast<double>(fmaxf(top_p, 0.f)) * static_cast<double>(mass));
        floor = cut_key<T, true>(w, floor, want < 1. ? 1ull : static_cast<unsigned long long>(want), weigh, hist, found);
    }
    const float* noise = a.noise + r * a.noise_stride;
    unsigned long long best = 0ull;   // score over complement of index
    float kept = 0.f;
    w.template each<4>(0, w.words, tid, blockDim.x, [&](const float* v, int j0) {
#pragma unroll
        for (int i = 0; i < kRowVec<T>; ++i) {
            const int j = j0 + i;
            const float x = weigh(v[i]);
            if (!(x > 0.f && x >= min_p) || entry_key(v[i], j) < floor || (greedy && x < 1.f)) continue;
            kept += x;
            const float score = greedy ? 1.f : x / noise[j];
            const unsigned long long key = static_cast<unsigned long long>(__float_as_uint(score)) << 32 |
                                           (0xffffffffu - static_cast<uint32_t>(j));
            if (score >= 0.f && key > best) best = key;
        }
    });
    best = block_reduce(best, MaxOp(), 0ull, red64);
    kept = block_reduce(kept, AddOp(), 0.f, red);
    if (tid == 0) {
        const int j = best ? key_index(best) : -1;
        a.tokens[r] = j;
        float lp = NAN;
        if (greedy) {
            lp = 0.f;
        } else if (j >= 0) {
            const float z = Elem<T>::to_f(w.row[j]);
            lp = (z == ms.m ? 0.f : (z - ms.m) / T0) - logf(kept);
        }
        a.logprobs[r] = lp;
    }
}

}  // namespace dwa

using namespace dwa;

extern "C" int dwa_top_logits(void* stream, const DwaLogitsDims* dims, const void* logits, int K, float temperature,
                              void* values, int32_t* indices, float* lse) {
    int rc = check_logits(dims, "top_logits");
    if (rc) return rc;
    if (K <= 0 || K > dims->V) return fail(DWA_ERR_INVALID_ARG, "top_logits: K must be in [1, V]");
    if (K > DWA_MAX_TOP) return fail(DWA_ERR_UNSUPPORTED, "top_logits: K > " + std::to_string(DWA_MAX_TOP));
    if (!(temperature > 0.f) || temperature > 1e30f)
        return fail(DWA_ERR_INVALID_ARG, "top_logits: temperature must be positive and finite");
    if (dims->rows == 0) return DWA_OK;
    if (!logits || !values || !indices || !lse) return fail(DWA_ERR_INVALID_ARG, "top_logits: a required pointer is NULL");
    if (reinterpret_cast<uintptr_t>(logits) % dtype_bytes(dims->dtype) ||
        reinterpret_cast<uintptr_t>(values) % dtype_bytes(dims->dtype))
        return fail(DWA_ERR_INVALID_ARG, "top_logits: a pointer is not aligned to its element");
    const TopArgs a = {logits, *dims, K, kLog2e / temperature, temperature, values, indices, lse};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const dim3 grid(static_cast<unsigned>(dims->rows));
    if (dims->dtype == DWA_BF16)
        DWA_TIMED("top_logits", st, (launch_pdl(top_logits_kernel<__nv_bfloat16>, grid, dim3(kSelThreads), 0, st, a)));
    else
        DWA_TIMED("top_logits", st, (launch_pdl(top_logits_kernel<float>, grid, dim3(kSelThreads), 0, st, a)));
    DWA_LAUNCH_CHECK("top_logits_kernel");
    ++g_launches_total;
    return DWA_OK;
}

extern "C" int dwa_sample_tokens(void* stream, const DwaLogitsDims* dims, const DwaSampleParams* params,
                                 const void* logits, const float* noise, int64_t noise_stride, int32_t* tokens,
                                 float* logprobs) {
    int rc = check_logits(dims, "sample_tokens");
    if (rc) return rc;
    if (!params) return fail(DWA_ERR_INVALID_ARG, "sample_tokens: params is NULL");
    if (noise_stride < 0) return fail(DWA_ERR_INVALID_ARG, "sample_tokens: noise_stride must not be negative");
    if (dims->rows == 0) return DWA_OK;
    if (!logits || !noise || !tokens || !logprobs)
        return fail(DWA_ERR_INVALID_ARG, "sample_tokens: a required pointer is NULL");
    if (reinterpret_cast<uintptr_t>(logits) % dtype_bytes(dims->dtype) || reinterpret_cast<uintptr_t>(noise) % 4)
        return fail(DWA_ERR_INVALID_ARG, "sample_tokens: a pointer is not aligned to its element");
    const SampleArgs a = {logits, *dims, noise, noise_stride, *params, tokens, logprobs};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const dim3 grid(static_cast<unsigned>(dims->rows));
    if (dims->dtype == DWA_BF16)
        DWA_TIMED("sample", st, (launch_pdl(sample_kernel<__nv_bfloat16>, grid, dim3(kSelThreads), 0, st, a)));
    else
        DWA_TIMED("sample", st, (launch_pdl(sample_kernel<float>, grid, dim3(kSelThreads), 0, st, a)));
    DWA_LAUNCH_CHECK("sample_kernel");
    ++g_launches_total;
    return DWA_OK;
}
