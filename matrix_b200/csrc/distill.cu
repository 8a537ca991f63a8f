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
// everything else is K entries a row.  A cluster of P CTAs holds a row in its
// shared memory (chunks of at most 72 KB, so that three CTAs share an SM and one
// loads while another writes), so the gradient reads nothing again.  One pass
// over the chunk keeps a running maximum and the sum of exp((z - max) / T) over
// the UNLISTED entries alone (a bitmap of the chunk tells which, one byte per
// 16-byte word of bf16): q_t as total minus listed would lose all its digits
// where the listed entries hold nearly everything.  Row sums are kept in fp32;
// what is left of a row (K terms and a few logarithms) is done in fp64, where
// differences of logarithms keep the digits that fp32 would round away.

#include <atomic>

#include "vocab_rows.cuh"

namespace dwa {

extern std::atomic<uint64_t> g_launches_total;

constexpr int kDistillThreads = 256;             // a CTA of a cluster that holds a row
constexpr int kStreamThreads = 512;              // a CTA that reads a row twice
constexpr int kRing = 5;                         // stages of two words a thread that such a CTA has in flight
constexpr int kDistillMaxCluster = 8;
constexpr int kDistillMaxParts = 64;             // warps that share a row
constexpr int kDistillPieces = 4;                // pieces in which a chunk arrives
constexpr int kDistillChunkBytes = 72 * 1024;    // three CTAs an SM
constexpr float kTailFloor = 5.9604645e-8f;      // 2^-24: what an fp32 log-sum-exp can tell from no tail
constexpr float kTailNone = 1.52587890625e-5f;   // 2^-16: a teacher's tail that may be its rounding alone

enum : int { kRowPlain = 0, kRowZero = 1, kRowBad = 2 };

// What the backward needs of a row.
struct RowState {
    float m, S;        // a reference and the sum of the student's weights relative to it (Ref)
    float log2_S;      // log2 S less its rounding to an integer, and
    float log2_S_int;  // that integer
    float of_tail;     // dL/dx of an unlisted entry over its q
    float L;           // the loss before its weight
    float t_hi, t_lo;  // log p_k = (t_k - t_hi) / T - t_lo
    float kind;        // kRowPlain, kRowZero (nothing to learn) or kRowBad
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
    float c;       // log2(e) / T
    double inv_T;
    int P, log_P;  // CTAs per row
    int room;      // words of the largest chunk
};

constexpr double kLn2 = 0.6931471805599453;

// log2(x) as an integer and a rest in [-0.5, 0.5], which fp32 holds to 2^-25.
__device__ __forceinline__ void log2_parts(float x, float& whole, float& rest) {
    const float l = log2f(x);
    whole = rintf(l);
    rest = fabsf(l) < INFINITY ? log2f(ldexpf(x, -static_cast<int>(whole))) : l;
}
// log(x) with the relative precision of fp32 also where x is 1 - y with a small y.
__device__ __forceinline__ float log_of_rest(float x, float y) { return x > 0.5f ? log1pf(-y) : logf(x); }

// dL/dx of a listed entry from its logits.
__device__ __forceinline__ float listed_grad(const RowState& s, const DistillArgs& a, float zk, float tk) {
    const Ref ref(s.m, a.c);
    const float q = ref.weight(zk, a.c) / s.S;
    const double lp = (static_cast<double>(tk) - s.t_hi) * a.inv_T - s.t_lo;
    if (!a.o.reverse) return q - (tk == -INFINITY ? 0.f : expf(static_cast<float>(lp)));
    if (q == 0.f) return 0.f;
    const double x = static_cast<double>(zk) * a.c, r = kLn2 * (x - ref.a(a.c) - s.log2_S_int - s.log2_S) - lp - s.L;
    return fabs(r) > 1e-14 * (fabs(x) + fabs(lp)) ? q * static_cast<float>(r) : 0.f;   // else the terms' rounding
}

// The unlisted entries' gradient of one row, word by word.
template <class T>
struct GradWriter {
    T* g;          // the row's gradient
    int V;
    bool fast;     // a plain row, and g has the phase of the logits
    int kind;
    Ref ref;
    float c, unl;

    __device__ __forceinline__ GradWriter(const RowWords<T>& w, T* g_, const RowState& s, const DistillArgs& a, float scale)
        : g(g_), V(w.V), kind(static_cast<int>(s.kind)), ref(s.m, a.c), c(a.c) {
        fast = kind == kRowPlain && (reinterpret_cast<uintptr_t>(g) - reinterpret_cast<uintptr_t>(w.row)) % 16 == 0;
        unl = kind == kRowPlain ? s.of_tail * scale / s.S : kind == kRowZero ? 0.f : NAN;
    }
    // any word
    __device__ __forceinline__ void operator()(uint4 x, int j0) const {
        constexpr int VEC = kRowVec<T>;
        uint64_t e[VEC / 2];
        float o[VEC];
        word_weights<T>(x, ref, c, e);
        unpair_word<T>(e, o);
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (j0 + i >= 0 && j0 + i < V) g[j0 + i] = Elem<T>::from_f(kind == kRowPlain ? o[i] * unl : unl);
    }
    // a whole word of a fast row
    __device__ __forceinline__ void whole(uint4 x, uint4* to) const {
        constexpr int VEC = kRowVec<T>;
        uint64_t e[VEC / 2];
        float o[VEC];
        word_weights<T>(x, ref, c, e);
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) e[i] = mul2(e[i], pair(unl, unl));
        unpair_word<T>(e, o);
        __stcs(to, pack<T>(o));
    }
};

// What the warps of a row's CTAs hand to all of them, a part each: a reference,
// the sum of the weights w of unlisted entries, and over listed entries the sum of
// w and, with x = log2(e) z / T ln 2, forward of p (log p - x), reverse of
// w (x - log p).
struct DistillParts {
    double L[kDistillMaxParts], S_l[kDistillMaxParts];
    float S_u[kDistillMaxParts], m[kDistillMaxParts];
    int bad[kDistillMaxCluster];
};

__device__ __forceinline__ void warp_sum_d(double& u, double& v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        u += __shfl_xor_sync(0xffffffffu, u, o);
        v += __shfl_xor_sync(0xffffffffu, v, o);
    }
}

// A row's state from its parts, and its loss: one warp.  P: the sum of the
// teacher's probabilities.
__device__ __forceinline__ double finish_row(RowState& s, const DistillParts& part, const DistillArgs& a, int valid,
                                             double P, int parts) {
    const int lane = threadIdx.x & 31;
    const bool one = lane < parts, two = lane + 32 < parts;
    const float m0 = one ? part.m[lane] : -INFINITY, m1 = two ? part.m[lane + 32] : -INFINITY;
    s.m = warp_max(fmaxf(m0, m1));
    const bool bad = __any_sync(0xffffffffu, lane < a.P && part.bad[lane]);
    const Ref ref(s.m, a.c);
    // a part without anything above -inf: its sums are 0 (NaN with a NaN)
    const float f0 = m0 > -INFINITY ? Ref(m0, a.c).rescale(ref, a.c) : 1.f;
    const float f1 = m1 > -INFINITY ? Ref(m1, a.c).rescale(ref, a.c) : 1.f;
    const float S_u = warp_sum((one ? f0 * part.S_u[lane] : 0.f) + (two ? f1 * part.S_u[lane + 32] : 0.f));
    double S_l = (one ? f0 * part.S_l[lane] : 0.) + (two ? f1 * part.S_l[lane + 32] : 0.);
    const double g0 = a.o.reverse ? f0 : 1.f, g1 = a.o.reverse ? f1 : 1.f;
    double L = (one ? g0 * part.L[lane] : 0.) + (two ? g1 * part.L[lane + 32] : 0.);
    warp_sum_d(S_l, L);
    const double S = S_u + S_l;
    s.S = static_cast<float>(S);
    log2_parts(s.S, s.log2_S_int, s.log2_S);
    // log q = x - log_S
    const double log_S = kLn2 * (ref.a(a.c) + s.log2_S_int + s.log2_S);
    if (a.o.reverse) L = (L - (S_l != 0. ? S_l * log_S : 0.)) / S;
    else L += P != 0. ? P * log_S : 0.;
    s.of_tail = 1.f;
    if (a.t_lse && valid < a.d.V) {
        const float p_t = fmaxf(static_cast<float>(1. - P), kTailFloor), q_t = S_u / s.S;
        if (q_t == 0.f) {
            if (!a.o.reverse && p_t > kTailNone) L = INFINITY;
            s.of_tail = 0.f;
        } else {
            const double r_t = static_cast<double>(log_of_rest(q_t, static_cast<float>(S_l) / s.S)) -
                               log_of_rest(p_t, static_cast<float>(P));
            L += a.o.reverse ? q_t * r_t : -p_t * r_t;
            s.of_tail = a.o.reverse ? static_cast<float>(r_t - L) : 1.f - p_t / q_t;
        }
    }
    const bool nothing = valid == 0 || (!a.t_lse && s.t_hi == -INFINITY);
    s.L = static_cast<float>(L);
    s.kind = bad ? kRowBad : nothing ? kRowZero : kRowPlain;
    return bad ? NAN : nothing ? 0. : L;
}

// A thread's words of a row on their way through shared memory, kRing stages of
// two words ahead, each pass right behind the one before.  Only the thread that
// copies a word reads it, so nothing but its own copies is waited for.
template <int NT>
struct WordRing {
    uint4* const slots;        // this thread's: 2 kRing of them, NT words apart
    const uint4* const src;    // its words, NT apart
    const int from, to;
    int left, next, put = 0, get = 0;

    __device__ __forceinline__ WordRing(uint4* slots_, const uint4* src_, int from_, int to_, int passes)
        : slots(slots_), src(src_), from(from_), to(to_), left(passes), next(from_) {}
    __device__ __forceinline__ void issue() {
        if (next >= to && left > 0) {
            --left;
            next = from;
        }
        if (left > 0 && next < to) {
            copy_async(slots + put * 2 * NT, src + next * NT);
            if (next + 1 < to) copy_async(slots + (put * 2 + 1) * NT, src + (next + 1) * NT);
            next += 2;
        }
        put = put + 1 == kRing ? 0 : put + 1;
        copy_commit();
    }
    template <class F>
    __device__ __forceinline__ void pass(F f) {   // f(word, its number) for all of them
        for (int k = from; k < to; k += 2) {
            copy_wait<kRing - 1>();
            const uint4* x = slots + get * 2 * NT;
            f(x[0], k);
            if (k + 1 < to) f(x[NT], k + 1);
            get = get + 1 == kRing ? 0 : get + 1;
            issue();
        }
    }
};

// The loss of a row, the state for a backward (a.state) and, with GRAD, the
// gradient of weight * L.  HOLD: a cluster of P CTAs holds the row in shared
// memory; else one CTA reads it, and for the gradient once more out of L2.
template <class T, bool GRAD, bool HOLD>
__global__ void __launch_bounds__(HOLD ? kDistillThreads : kStreamThreads, HOLD ? 3 : 2)
    distill_fwd_kernel(const __grid_constant__ DistillArgs a) {
    namespace cg = cooperative_groups;
    constexpr int NT = HOLD ? kDistillThreads : kStreamThreads, WARPS = NT / 32;
    constexpr int VEC = kRowVec<T>, MOST = DWA_MAX_TOP / NT;
    extern __shared__ __align__(16) uint4 data[];
    __shared__ DistillParts part;
    __shared__ double redd[33];
    __shared__ float redf[33];
    __shared__ RowState row_state;
    __shared__ int bad, valid;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = a.o.K, V = a.d.V;
    const uint32_t r = blockIdx.x >> a.log_P;
    const int p = blockIdx.x & (a.P - 1);
    uint32_t* bits = reinterpret_cast<uint32_t*>(data + (HOLD ? a.room : 2 * kRing * NT));
    if (a.P > 1) cluster_arrive_relaxed();
    if (tid == 0) bad = valid = 0;
    pdl_enter();
    // the teacher's loads first, then the chunk's copies, which they would wait behind
    const int64_t rK = static_cast<int64_t>(r) * K;
    int j[MOST];
    float t[MOST];
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
        const int k = tid + i * NT;
        j[i] = -1;
        t[i] = -INFINITY;
        if (k < K) {
            j[i] = a.idx[rK + k];
            t[i] = load_elem(a.t, rK + k, a.o.teacher_dtype);
        }
    }
    const float weight = a.weights ? a.weights[r] : 1.f, t_lse = a.t_lse ? a.t_lse[r] : 0.f;
    const RowWords<T> w(static_cast<const T*>(a.z) + row_offset(a.d, r), V);
    const Chunk ch(w.words, p, a.log_P);
    const int n = ch.hi - ch.lo;
    T* g = GRAD ? static_cast<T*>(a.g) + static_cast<int64_t>(r) * V : nullptr;
    // the chunk, in pieces: every thread copies the words that it will look at
    int from, to;
    w.own_whole(ch.lo, ch.hi, tid, NT, from, to);
    uint4* const own_words = data + tid;
    float z[MOST];   // the listed entries' logits
    const auto piece = [&](int i) { return from + (to - from) * i / kDistillPieces; };
    const uint4* const src = reinterpret_cast<const uint4*>(w.row + w.first(ch.lo + tid));
    WordRing<NT> ring(own_words, src, from, to, GRAD ? 2 : 1);
    if constexpr (HOLD) {
#pragma unroll
        for (int i = 0; i < kDistillPieces; ++i) {
            const int end = piece(i + 1);
#pragma unroll 4
            for (int k = piece(i); k < end; ++k) copy_async(own_words + k * NT, src + k * NT);
            copy_commit();
        }
    } else {
#pragma unroll
        for (int i = 0; i < kRing; ++i) ring.issue();
#pragma unroll
        for (int i = 0; i < MOST; ++i) z[i] = j[i] >= 0 && j[i] < V ? Elem<T>::to_f(w.row[j[i]]) : -INFINITY;
    }
    for (int i = tid; i < (n * VEC + 127) / 128; i += NT)
        reinterpret_cast<uint4*>(bits)[i] = make_uint4(0u, 0u, 0u, 0u);
    __syncthreads();
    RowState s = {};
    if (weight == 0.f) {   // a row left out, whatever it holds
        s.kind = kRowZero;
        if (p == 0 && tid == 0) {
            a.loss[r] = 0.f;
            if (a.state) a.state[r] = s;
        }
        copy_wait<0>();
        if constexpr (GRAD) {
            const GradWriter<T> write(w, g, s, a, 0.f);
            for (int i = ch.lo + tid; i < ch.hi; i += NT) write(make_uint4(0u, 0u, 0u, 0u), w.first(i));
        }
        if (a.P > 1) cluster_wait();
        return;
    }
    // the teacher: every CTA all of it, the places of the entries in its chunk
    int mine = 0, at[MOST];
    float t_top = -INFINITY, prob[MOST];
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
        at[i] = -1;
        if (j[i] >= V) bad = 1;
        if (j[i] < 0 || j[i] >= V) {
            t[i] = -INFINITY;
            continue;
        }
        ++mine;
        const int b = j[i] + w.shift - ch.lo * VEC;
        if (b >= 0 && b < n * VEC) {
            at[i] = b;
            if (atomicOr(&bits[b >> 5], 1u << (b & 31)) & (1u << (b & 31))) bad = 1;
        }
        t_top = fmaxf(t_top, t[i]);
    }
    if (mine) atomicAdd(&valid, mine);
    if (a.t_lse) {
        s.t_lo = t_lse;
    } else {
        s.t_hi = block_reduce(t_top, MaxOp(), -INFINITY, redf);
        double sum = 0.;
#pragma unroll
        for (int i = 0; i < MOST; ++i)
            if (t[i] > -INFINITY) sum += expf(static_cast<float>((static_cast<double>(t[i]) - s.t_hi) * a.inv_T));
        s.t_lo = logf(static_cast<float>(block_reduce(sum, AddOp(), 0., redd)));
    }
    const auto log_p = [&](float x) { return (static_cast<double>(x) - s.t_hi) * a.inv_T - s.t_lo; };
    double P = 0.;
#pragma unroll
    for (int i = 0; i < MOST; ++i) {
        prob[i] = t[i] == -INFINITY ? 0.f : expf(static_cast<float>(log_p(t[i])));
        if (tid + i * NT < K) P += prob[i];
    }
    P = block_reduce(P, AddOp(), 0., redd);   // its barriers also order the bitmap
    // one pass: the sum of the weights of unlisted entries
    MaxSum ms;
    const uint8_t* byte = reinterpret_cast<const uint8_t*>(bits);
    const auto add_word = [&](uint4 x, int k) {
        const float top = word_max<T>(x);
        const uint32_t listed = VEC == 8 ? byte[k] : (byte[k >> 1] >> (4 * (k & 1))) & 15u;
        if (!ms.covers(top)) {
            ms.raise(top, a.c);
            if (top != top) ms.poison();
            if (ms.ref.m == -INFINITY) return;
        }
        uint64_t e[VEC / 2];
        word_weights<T>(x, ms.ref, a.c, e);
        if (listed != 0u) {
            float f[VEC];
            unpair_word<T>(e, f);
#pragma unroll
            for (int v = 0; v < VEC; v += 2)
                e[v / 2] = pair((listed >> v) & 1u ? 0.f : f[v], (listed >> v) & 2u ? 0.f : f[v + 1]);
        }
        ms.s2 = add2(ms.s2, sum_pairs<T>(e));
    };
    w.edges(ch.lo, ch.hi, tid, [&](uint4 x, int j0) {
        const int k = (j0 + w.shift) / VEC - ch.lo;
        if constexpr (HOLD) data[k] = x;
        add_word(x, k);
    });
    if constexpr (HOLD) {
        const auto add = [&](int i) {
            const int end = piece(i + 1);
#pragma unroll 2
            for (int k = piece(i); k < end; ++k) add_word(own_words[k * NT], tid + k * NT);
        };
        static_assert(kDistillPieces == 4, "one wait a piece");
        copy_wait<3>();
        add(0);
        copy_wait<2>();
        add(1);
        copy_wait<1>();
        add(2);
        copy_wait<0>();
        add(3);
        __syncthreads();   // the listed entries may be other threads' words
#pragma unroll
        for (int i = 0; i < MOST; ++i)
            z[i] = at[i] >= 0 ? Elem<T>::to_f(reinterpret_cast<const T*>(data)[at[i]]) : -INFINITY;
    } else {
        ring.pass([&](uint4 x, int k) { add_word(x, tid + k * NT); });
    }
    // the warp's part: what it summed, and its listed entries of this chunk
    float top = ms.ref.m;
#pragma unroll
    for (int i = 0; i < MOST; ++i) top = fmaxf(top, z[i]);
    const Ref ref(warp_max(top), a.c);
    const float S_u = warp_sum(ms.at(ref, a.c));
    double S_l = 0., L = 0.;
    if (warp * 32 < K) {
#pragma unroll
        for (int i = 0; i < MOST; ++i) {
            if (at[i] < 0) continue;
            const double lp = log_p(t[i]), x = kLn2 * a.c * z[i];
            const float e = z[i] == -INFINITY ? 0.f : ref.weight(z[i], a.c);   // the reference may be -inf too
            S_l += e;
            if (a.o.reverse) L += e != 0.f ? e * (x - lp) : 0.;
            else L += prob[i] != 0.f ? prob[i] * (lp - x) : 0.;
        }
        warp_sum_d(S_l, L);
    }
    if (a.P > 1) cluster_wait();   // every CTA of the cluster has started
    if (lane < a.P) {              // lane q: to CTA q
        DistillParts& to_q = *cg::this_cluster().map_shared_rank(&part, lane);
        const int i = p * WARPS + warp;
        to_q.m[i] = ref.m;
        to_q.S_u[i] = S_u;
        to_q.S_l[i] = S_l;
        to_q.L[i] = L;
        if (warp == 0) to_q.bad[p] = bad;
    }
    if (a.P > 1) cg::this_cluster().sync();
    else __syncthreads();
    if (!GRAD && p != 0) return;
    if (warp == 0) {
        const double loss = finish_row(s, part, a, valid, P, a.P * WARPS);
        if (lane == 0) row_state = s;
        if (p == 0 && lane == 0) {
            if (s.kind == kRowBad) raise_status(a.status, DWA_STATUS_BAD_TOKEN);
            a.loss[r] = static_cast<float>(loss * weight);
            if (a.state) a.state[r] = s;
        }
    }
    if constexpr (GRAD) {
        __syncthreads();
        s = row_state;
        const float scale = weight * static_cast<float>(a.inv_T);
        const GradWriter<T> write(w, g, s, a, scale);
        if (write.fast) {
            uint4* const to_g = reinterpret_cast<uint4*>(g + w.first(ch.lo + tid));
            if constexpr (HOLD) {
#pragma unroll 4
                for (int k = from; k < to; ++k) write.whole(own_words[k * NT], to_g + k * NT);
            } else {
                ring.pass([&](uint4 x, int k) { write.whole(x, to_g + k * NT); });
            }
            w.edges(ch.lo, ch.hi, tid, write);
        } else {
            if constexpr (HOLD) {
                for (int k = tid; k < n; k += NT) write(data[k], w.first(ch.lo + k));
            } else {
                ring.pass([&](uint4 x, int k) { write(x, w.first(tid + k * NT)); });
                w.edges(ch.lo, ch.hi, tid, write);
            }
        }
        if (s.kind != kRowPlain) return;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < MOST; ++i)
            if (at[i] >= 0) g[j[i]] = Elem<T>::from_f(listed_grad(s, a, z[i], t[i]) * scale);
    }
}

// The gradient from a saved state: P CTAs per row, each its words.  g may be the
// logits' own memory: a listed entry is read before its word is written.
template <class T>
__global__ void __launch_bounds__(kDistillThreads) distill_bwd_kernel(const __grid_constant__ DistillArgs a) {
    pdl_enter();
    constexpr int VEC = kRowVec<T>;
    extern __shared__ float zk[];
    const int tid = threadIdx.x, K = a.o.K, V = a.d.V;
    const uint32_t r = blockIdx.x >> a.log_P;
    const RowWords<T> w(static_cast<const T*>(a.z) + row_offset(a.d, r), V);
    const Chunk ch(w.words, blockIdx.x & (a.P - 1), a.log_P);
    const int32_t* idx = a.idx + static_cast<int64_t>(r) * K;
    const RowState s = a.state[r];
    const bool plain = s.kind == kRowPlain;
    const auto here = [&](int j) { return j >= 0 && (j + w.shift) / VEC >= ch.lo && (j + w.shift) / VEC < ch.hi; };
    if (plain) {
        for (int k = tid; k < K; k += kDistillThreads)
            if (here(idx[k])) zk[k] = Elem<T>::to_f(w.row[idx[k]]);
        __syncthreads();
    }
    const float scale = (a.weights ? a.weights[r] : 1.f) * a.g_loss[r] * static_cast<float>(a.inv_T);
    T* g = static_cast<T*>(a.g) + static_cast<int64_t>(r) * V;
    const GradWriter<T> write(w, g, s, a, scale);
    if (write.fast) {
        w.template each_whole<4>(ch.lo, ch.hi, tid, kDistillThreads, [&](uint4 x, int j0, int) {
            write.whole(x, reinterpret_cast<uint4*>(g + j0));
        });
        w.edges(ch.lo, ch.hi, tid, write);
    } else {
        w.template each<1>(ch.lo, ch.hi, tid, kDistillThreads, [&](uint4 x, int j0, int) { write(x, j0); });
    }
    if (!plain) return;
    __syncthreads();
    for (int k = tid; k < K; k += kDistillThreads)
        if (here(idx[k]))
            g[idx[k]] = Elem<T>::from_f(listed_grad(s, a, zk[k], load_elem(a.t, static_cast<int64_t>(r) * K + k, a.o.teacher_dtype)) * scale);
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
    if (d->rows >= (int64_t(1) << 28)) return fail(DWA_ERR_UNSUPPORTED, w + ": rows >= 2^28");
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

// CTAs per row that hold it: enough that a chunk leaves room for three CTAs an SM
// (or fits at all), more while the launch is short of two CTAs an SM and chunks
// stay above 16 KB.
static int log_ctas_per_row(const DwaLogitsDims& d) {
    const int64_t bytes = static_cast<int64_t>(d.V) * dtype_bytes(d.dtype);
    int l = 0;
    while (1 << l < kDistillMaxCluster &&
           (bytes > kDistillChunkBytes << l || (d.rows << l < 2 * tc::sm_count() && bytes > 32 * 1024 << l)))
        ++l;
    return l;
}

template <class T, bool GRAD, bool HOLD>
static int launch_fwd_as(cudaStream_t st, DistillArgs a) {
    constexpr int VEC = kRowVec<T>, NT = HOLD ? kDistillThreads : kStreamThreads;
    a.log_P = HOLD ? log_ctas_per_row(a.d) : 0;
    a.P = 1 << a.log_P;
    a.room = (a.d.V + 2 * VEC - 2) / VEC / a.P + 1;
    const size_t sh = static_cast<size_t>(HOLD ? a.room : 2 * kRing * NT) * 16 + (static_cast<size_t>(a.room) * VEC + 127) / 128 * 16;
    if (int rc = allow_smem(distill_fwd_kernel<T, GRAD, HOLD>, sh)) return rc;
    DWA_TIMED("distill_fwd", st,
              (launch_pdl_cluster(distill_fwd_kernel<T, GRAD, HOLD>, dim3(static_cast<unsigned>(a.d.rows * a.P)), dim3(NT),
                                  sh, st, dim3(a.P), a)));
    DWA_LAUNCH_CHECK("distill_fwd_kernel");
    ++g_launches_total;
    return DWA_OK;
}

template <class T, bool GRAD>
static int launch_fwd(cudaStream_t st, const DistillArgs& a) {
    if (a.d.rows >= 2 * tc::sm_count()) return launch_fwd_as<T, GRAD, false>(st, a);
    return launch_fwd_as<T, GRAD, true>(st, a);
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
                           kLog2e / opts->temperature, 1. / opts->temperature, 1, 0, 0};
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
    const int log_P = log_ctas_per_row(*dims);
    const DistillArgs a = {logits, *dims, *opts, teacher_logits, teacher_indices, teacher_lse, weights, nullptr,
                           reinterpret_cast<RowState*>(const_cast<float*>(state)), g_loss, g_logits, nullptr,
                           kLog2e / opts->temperature, 1. / opts->temperature, 1 << log_P, log_P, 0};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const size_t sh = static_cast<size_t>(opts->K) * 4;
    const dim3 grid(static_cast<unsigned>(dims->rows << log_P));
    if (dims->dtype == DWA_BF16)
        DWA_TIMED("distill_bwd", st,
                  (launch_pdl(distill_bwd_kernel<__nv_bfloat16>, grid, dim3(kDistillThreads), sh, st, a)));
    else
        DWA_TIMED("distill_bwd", st, (launch_pdl(distill_bwd_kernel<float>, grid, dim3(kDistillThreads), sh, st, a)));
    DWA_LAUNCH_CHECK("distill_bwd_kernel");
    ++g_launches_total;
    return DWA_OK;
}
