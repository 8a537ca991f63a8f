// Distillation of a student's logits from the top logits of a teacher.
//
// For one row, with the student's logits z [V], the listed entries i_k with the
// teacher's logits t_k (k < K), and temperature T:
//   q = softmax(z / T),  q_k = q[i_k]
//   no tail:  p = softmax(t / T) over the listed entries
//   tail:     p_k = exp(t_k / T - lse) with the teacher's log-sum-exp, and one
//             class for all other entries: p_t = max(1 - sum p, 2^-24),
//             q_t = sum of the unlisted q
//   forward:  L = sum p (log p - log q);  dL/d(z_j / T) = q_j - p_j on listed
//             entries, q_j (1 - p_t / q_t) (no tail: q_j) on the others
//   reverse:  L = sum q (log q - log p);  with r = log q - log p:
//             q_k (r_k - L) on listed entries, q_j (r_t - L) on the others
// The gradient is thus one coefficient times q on unlisted entries, and K
// entries set apart.
//
// Bound: HBM.  The loss has to read the row once, the gradient to write it once;
// everything else is K entries a row.  The forward keeps a running maximum and
// the sum of exp((z - max) / T) over the UNLISTED entries alone (a bitmap of the
// row in shared memory tells which, one byte per 16-byte word of bf16): q_t as
// total minus listed would lose all its digits where the listed entries hold
// nearly everything.  Row sums are kept in fp32, what is left of a row (K terms
// and a few logarithms) is done in fp64, where differences of logarithms keep
// the digits that fp32 would round away.

#include <atomic>

#include "vocab_rows.cuh"

namespace dwa {

extern std::atomic<uint64_t> g_launches_total;

constexpr int kDistillThreads = 512;
constexpr float kTailFloor = 5.9604645e-8f;      // 2^-24: what an fp32 log-sum-exp can tell from no tail
constexpr float kTailNone = 1.52587890625e-5f;   // 2^-16: a teacher's tail that may be its rounding alone

enum : int { kRowPlain = 0, kRowZero = 1, kRowBad = 2 };

// What the backward needs of a row.
struct RowState {
    float m, S;        // the student's maximum and sum of exp((z - m) / T)
    float of_tail;     // dL/dx of an unlisted entry over its q
    float L;           // the loss before its weight
    float t_hi, t_lo;  // log p_k = (t_k - t_hi) / T - t_lo
    float kind;        // kRowPlain, kRowZero (nothing to learn) or kRowBad
    float unused;
};
static_assert(sizeof(RowState) == DWA_DISTILL_STATE_FLOATS * sizeof(float), "layout of the saved row state");

struct DistillArgs {
    const void* z;
    DwaLogitsDims d;
    DwaDistillDims o;
    const void* t;
    const int32_t* idx;
    const float* t_lse;
    const float* weights;
    float* loss;
    RowState* state;
    const float* g_loss;
    void* g;
    uint32_t* status;
    float c;   // log2(e) / T
};

// dL/dx of listed entry k, from its logits.
__device__ __forceinline__ float listed_grad(const RowState& s, const DistillArgs& a, float zk, float tk) {
    const float q = exp2_fast((zk - s.m) * a.c) / s.S;
    const double T = a.o.temperature;
    const double lp = (static_cast<double>(tk) - s.t_hi) / T - s.t_lo;
    if (!a.o.reverse) return q - (tk == -INFINITY ? 0.f : expf(static_cast<float>(lp)));
    if (q == 0.f) return 0.f;
    const double lq = (static_cast<double>(zk) - s.m) / T - log(static_cast<double>(s.S));
    return q * static_cast<float>(lq - lp - s.L);
}

// The gradient of one row into g [V]: the unlisted coefficient times q over the
// whole row, then the listed entries.  `zk`, `tk` (shared memory) were read
// before, so g may be the logits' own memory.
template <class T>
__device__ __forceinline__ void write_grad(const RowWords<T>& w, T* g, const RowState& s, const DistillArgs& a,
                                           float scale, const float* zk, const float* tk, const int32_t* idx) {
    constexpr int VEC = kRowVec<T>;
    const int tid = threadIdx.x, n = blockDim.x;
    const int kind = static_cast<int>(s.kind);
    const float unl = kind == kRowPlain ? s.of_tail * scale / s.S : kind == kRowZero ? 0.f : NAN;
    const bool same = (reinterpret_cast<uintptr_t>(g) - reinterpret_cast<uintptr_t>(w.row)) % 16 == 0;
    w.template each<4>(0, w.words, tid, n, [&](uint4 x, int j0, int) {
        float o[VEC];
        word_exp<T>(x, s.m, a.c, o);
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[i] = kind == kRowPlain ? o[i] * unl : unl;
        if (same && j0 >= 0 && j0 + VEC <= w.V) {
            *reinterpret_cast<uint4*>(g + j0) = pack<T>(o);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (j0 + i >= 0 && j0 + i < w.V) g[j0 + i] = Elem<T>::from_f(o[i]);
        }
    });
    if (kind != kRowPlain) return;
    __syncthreads();
    for (int k = tid; k < a.o.K; k += n)
        if (idx[k] >= 0) g[idx[k]] = Elem<T>::from_f(listed_grad(s, a, zk[k], tk[k]) * scale);
}

// One CTA per row: the loss, the state for a backward (a.state) and, with GRAD,
// the gradient of weight * L (the row is read again, out of L2).
template <class T, bool GRAD>
__global__ void __launch_bounds__(kDistillThreads) distill_fwd_kernel(DistillArgs a) {
    pdl_enter();
    constexpr int VEC = kRowVec<T>;
    extern __shared__ float sm[];
    __shared__ float redf[33];
    __shared__ double redd[33];
    __shared__ int bad, valid;
    const int tid = threadIdx.x, n = blockDim.x, K = a.o.K, V = a.d.V;
    const int64_t r = blockIdx.x;
    const RowWords<T> w(static_cast<const T*>(a.z) + row_offset(a.d, r), V);
    T* g = GRAD ? static_cast<T*>(a.g) + r * V : nullptr;
    const int32_t* idx = a.idx + r * K;
    float* zk = sm;
    float* tk = zk + K;
    uint32_t* bits = reinterpret_cast<uint32_t*>(tk + K);
    const float weight = a.weights ? a.weights[r] : 1.f;
    RowState s = {};
    if (weight == 0.f) {   // a row left out: its logits and teacher are not looked at
        s.kind = kRowZero;
        if (tid == 0) {
            a.loss[r] = 0.f;
            if (a.state) a.state[r] = s;
        }
        if constexpr (GRAD) write_grad(w, g, s, a, 0.f, zk, tk, idx);
        return;
    }
    for (int i = tid; i < (w.words * VEC + 31) / 32; i += n) bits[i] = 0u;
    if (tid == 0) bad = valid = 0;
    __syncthreads();
    int mine = 0;
    for (int k = tid; k < K; k += n) {
        const int j = idx[k];
        float z = -INFINITY, t = -INFINITY;
        if (j >= V) {
            bad = 1;
        } else if (j >= 0) {
            const int b = j + w.shift;
            if (atomicOr(&bits[b >> 5], 1u << (b & 31)) & (1u << (b & 31))) bad = 1;
            z = Elem<T>::to_f(w.row[j]);
            t = load_elem(a.t, r * K + k, a.o.teacher_dtype);
            ++mine;
        }
        zk[k] = z;
        tk[k] = t;
    }
    if (mine) atomicAdd(&valid, mine);
    __syncthreads();

    // one pass: the row's maximum, and the sum over unlisted entries
    MaxSum ms;
    w.template each<4>(0, w.words, tid, n, [&](uint4 x, int j0, int) {
        ms.raise(word_max<T>(x), a.c);
        float e[VEC];
        word_exp<T>(x, ms.m, a.c, e);
        const int b = j0 + w.shift;
        const uint32_t listed = bits[b >> 5] >> (b & 31) & ((1u << VEC) - 1u);
        if (listed == 0u && ms.m > -INFINITY) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) ms.s += e[i];
        } else if (ms.m > -INFINITY) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) ms.s += (listed >> i) & 1u ? 0.f : e[i];
        }
    });
    s.m = block_reduce(ms.m, MaxOp(), -INFINITY, redf);
    const float S_u = block_reduce(ms.at(s.m, a.c), AddOp(), 0.f, redf);

    // the listed entries
    const double T0 = a.o.temperature;
    float S_l = 0.f;
    for (int k = tid; k < K; k += n)
        if (idx[k] >= 0) S_l += exp2_fast((zk[k] - s.m) * a.c);
    S_l = block_reduce(S_l, AddOp(), 0.f, redf);
    s.S = S_u + S_l;
    const double log_S = log(static_cast<double>(S_u) + S_l);
    if (a.t_lse) {
        s.t_hi = 0.f;
        s.t_lo = a.t_lse[r];
    } else {
        float top = -INFINITY;
        for (int k = tid; k < K; k += n) top = fmaxf(top, tk[k]);
        s.t_hi = block_reduce(top, MaxOp(), -INFINITY, redf);
        double sum = 0.;
        for (int k = tid; k < K; k += n)
            if (idx[k] >= 0) sum += expf(static_cast<float>((static_cast<double>(tk[k]) - s.t_hi) / T0));
        s.t_lo = static_cast<float>(log(block_reduce(sum, AddOp(), 0., redd)));
    }
    double P = 0., L = 0.;
    for (int k = tid; k < K; k += n) {
        if (idx[k] < 0) continue;
        const double lp = (static_cast<double>(tk[k]) - s.t_hi) / T0 - s.t_lo;
        const double lq = (static_cast<double>(zk[k]) - s.m) / T0 - log_S;
        const float p = tk[k] == -INFINITY ? 0.f : expf(static_cast<float>(lp));
        P += p;
        if (a.o.reverse) {
            const float q = exp2_fast((zk[k] - s.m) * a.c) / s.S;
            if (q != 0.f) L += q * (lq - lp);
        } else if (p != 0.f) {
            L += p * (lp - lq);
        }
    }
    P = block_reduce(P, AddOp(), 0., redd);
    L = block_reduce(L, AddOp(), 0., redd);
    const bool nothing = valid == 0 || (!a.t_lse && s.t_hi == -INFINITY);
    s.of_tail = 1.f;
    if (a.t_lse && valid < V) {
        const double p_t = fmax(1. - P, static_cast<double>(kTailFloor));
        const double q_t = S_u / (static_cast<double>(S_u) + S_l);
        if (q_t == 0.) {
            if (!a.o.reverse && p_t > kTailNone) L = INFINITY;
            s.of_tail = 0.f;
        } else {
            const double r_t = log(q_t) - log(p_t);
            L += a.o.reverse ? q_t * r_t : -p_t * r_t;
            s.of_tail = static_cast<float>(a.o.reverse ? r_t - L : 1. - p_t / q_t);
        }
    }
    s.L = static_cast<float>(L);
    s.kind = bad ? kRowBad : nothing ? kRowZero : kRowPlain;
    if (tid == 0) {
        if (bad) raise_status(a.status, DWA_STATUS_BAD_TOKEN);
        a.loss[r] = bad ? NAN : nothing ? 0.f : static_cast<float>(L * weight);
        if (a.state) a.state[r] = s;
    }
    if constexpr (GRAD) write_grad(w, g, s, a, weight / a.o.temperature, zk, tk, idx);
}

// The gradient from a saved state: one CTA per row.
template <class T>
__global__ void __launch_bounds__(kDistillThreads) distill_bwd_kernel(DistillArgs a) {
    pdl_enter();
    extern __shared__ float sm[];
    const int tid = threadIdx.x, n = blockDim.x, K = a.o.K, V = a.d.V;
    const int64_t r = blockIdx.x;
    const RowWords<T> w(static_cast<const T*>(a.z) + row_offset(a.d, r), V);
    const int32_t* idx = a.idx + r * K;
    float* zk = sm;
    float* tk = zk + K;
    const RowState s = a.state[r];
    if (s.kind == kRowPlain) {
        for (int k = tid; k < K; k += n) {
            if (idx[k] < 0) continue;
            zk[k] = Elem<T>::to_f(w.row[idx[k]]);
            tk[k] = load_elem(a.t, r * K + k, a.o.teacher_dtype);
        }
    }
    __syncthreads();
    const float weight = (a.weights ? a.weights[r] : 1.f) * a.g_loss[r];
    write_grad(w, static_cast<T*>(a.g) + r * V, s, a, weight / a.o.temperature, zk, tk, idx);
}

int check_logits(const DwaLogitsDims* d, const char* what) {
    const std::string w(what);
    if (!d) return fail(DWA_ERR_INVALID_ARG, w + ": dims is NULL");
    if (d->dtype != DWA_F32 && d->dtype != DWA_BF16)
        return fail(DWA_ERR_INVALID_ARG, w + ": dtype must be DWA_F32 or DWA_BF16");
    if (d->rows < 0 || d->V <= 0 || d->rows_inner <= 0)
        return fail(DWA_ERR_INVALID_ARG, w + ": rows must not be negative, V and rows_inner be positive");
    if (d->stride_outer < 0 || d->stride_inner < 0)
        return fail(DWA_ERR_INVALID_ARG, w + ": strides must not be negative");
    if (d->V > DWA_MAX_VOCAB) return fail(DWA_ERR_UNSUPPORTED, w + ": V > " + std::to_string(DWA_MAX_VOCAB));
    if (d->rows >= (int64_t(1) << 31)) return fail(DWA_ERR_UNSUPPORTED, w + ": rows >= 2^31");
    return DWA_OK;
}

static int check_distill(const DwaLogitsDims* d, const DwaDistillDims* o, const float* t_lse) {
    int rc = check_logits(d, "distill");
    if (rc) return rc;
    if (!o) return fail(DWA_ERR_INVALID_ARG, "distill: options are NULL");
    if (o->K <= 0 || o->K > d->V) return fail(DWA_ERR_INVALID_ARG, "distill: K must be in [1, V]");
    if (o->K > DWA_MAX_TOP) return fail(DWA_ERR_UNSUPPORTED, "distill: K > " + std::to_string(DWA_MAX_TOP));
    if (o->teacher_dtype != DWA_F32 && o->teacher_dtype != DWA_BF16)
        return fail(DWA_ERR_INVALID_ARG, "distill: teacher_dtype must be DWA_F32 or DWA_BF16");
    if (!(o->temperature > 0.f) || o->temperature > 1e30f)
        return fail(DWA_ERR_INVALID_ARG, "distill: temperature must be positive and finite");
    if (o->reverse && !t_lse)
        return fail(DWA_ERR_INVALID_ARG, "distill: the reverse divergence needs the teacher's log-sum-exp");
    return DWA_OK;
}

static int check_workspace(const void* ws, size_t bytes) {
    if (!ws || reinterpret_cast<uintptr_t>(ws) % 256 != 0)
        return fail(DWA_ERR_WORKSPACE, "workspace must be non-NULL and 256-byte aligned");
    if (bytes < dwa_distill_workspace_bytes()) return fail(DWA_ERR_WORKSPACE, "workspace too small");
    return DWA_OK;
}

static bool misaligned(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % dtype_bytes(dtype) != 0; }

template <class K>
static int allow_smem(K kernel, size_t bytes) {
    if (bytes > 48 * 1024)
        DWA_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)));
    return DWA_OK;
}

template <class T, bool GRAD>
static int launch_fwd(cudaStream_t st, const DistillArgs& a) {
    const size_t sh = static_cast<size_t>(a.o.K) * 8 + align_up(static_cast<size_t>(a.d.V) / 8 + 8, 16);
    if (int rc = allow_smem(distill_fwd_kernel<T, GRAD>, sh)) return rc;
    DWA_TIMED("distill_fwd", st, (launch_pdl(distill_fwd_kernel<T, GRAD>, dim3(static_cast<unsigned>(a.d.rows)),
                                             dim3(kDistillThreads), sh, st, a)));
    DWA_LAUNCH_CHECK("distill_fwd_kernel");
    ++g_launches_total;
    return DWA_OK;
}

}  // namespace dwa

using namespace dwa;

extern "C" size_t dwa_distill_workspace_bytes(void) { return 256; }

extern "C" int dwa_distill_fwd(void* stream, const DwaLogitsDims* dims, const DwaDistillDims* opts, const void* logits,
                               const void* teacher_logits, const int32_t* teacher_indices, const float* teacher_lse,
                               const float* weights, float* loss, float* state, void* g_logits, void* workspace,
                               size_t workspace_bytes) {
    int rc = check_distill(dims, opts, teacher_lse);
    if (rc) return rc;
    if (dims->rows == 0) return DWA_OK;
    if (!logits || !teacher_logits || !teacher_indices || !loss)
        return fail(DWA_ERR_INVALID_ARG, "distill: a required pointer is NULL");
    if (misaligned(logits, dims->dtype) || misaligned(g_logits, dims->dtype) ||
        misaligned(teacher_logits, opts->teacher_dtype))
        return fail(DWA_ERR_INVALID_ARG, "distill: a pointer is not aligned to its element");
    if ((rc = check_workspace(workspace, workspace_bytes))) return rc;
    const DistillArgs a = {logits, *dims, *opts, teacher_logits, teacher_indices, teacher_lse, weights, loss,
                           reinterpret_cast<RowState*>(state), nullptr, g_logits, static_cast<uint32_t*>(workspace),
                           kLog2e / opts->temperature};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dims->dtype == DWA_BF16)
        return g_logits ? launch_fwd<__nv_bfloat16, true>(st, a) : launch_fwd<__nv_bfloat16, false>(st, a);
    return g_logits ? launch_fwd<float, true>(st, a) : launch_fwd<float, false>(st, a);
}

extern "C" int dwa_distill_bwd(void* stream, const DwaLogitsDims* dims, const DwaDistillDims* opts, const void* logits,
                               const void* teacher_logits, const int32_t* teacher_indices, const float* teacher_lse,
                               const float* weights, const float* state, const float* g_loss, void* g_logits) {
    int rc = check_distill(dims, opts, teacher_lse);
    if (rc) return rc;
    if (dims->rows == 0) return DWA_OK;
    if (!logits || !teacher_logits || !teacher_indices || !state || !g_loss || !g_logits)
        return fail(DWA_ERR_INVALID_ARG, "distill: a required pointer is NULL");
    if (misaligned(logits, dims->dtype) || misaligned(g_logits, dims->dtype) ||
        misaligned(teacher_logits, opts->teacher_dtype))
        return fail(DWA_ERR_INVALID_ARG, "distill: a pointer is not aligned to its element");
    const DistillArgs a = {logits, *dims, *opts, teacher_logits, teacher_indices, teacher_lse, weights, nullptr,
                           reinterpret_cast<RowState*>(const_cast<float*>(state)), g_loss, g_logits, nullptr,
                           kLog2e / opts->temperature};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const size_t sh = static_cast<size_t>(opts->K) * 8;
    const dim3 grid(static_cast<unsigned>(dims->rows));
    if (dims->dtype == DWA_BF16)
        DWA_TIMED("distill_bwd", st,
                  (launch_pdl(distill_bwd_kernel<__nv_bfloat16>, grid, dim3(kDistillThreads), sh, st, a)));
    else
        DWA_TIMED("distill_bwd", st, (launch_pdl(distill_bwd_kernel<float>, grid, dim3(kDistillThreads), sh, st, a)));
    DWA_LAUNCH_CHECK("distill_bwd_kernel");
    ++g_launches_total;
    return DWA_OK;
}
