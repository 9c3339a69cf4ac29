// Operators on a model's output distribution: log probabilities of given
// tokens with entropy and top alternatives, and the distillation loss from a
// teacher's top log probabilities; forward and backward.
//
// Mathematics, for one row x of V logits at temperature T:
//   m = max x, d_j = (x_j - m) / T, s = sum e^{d_j}, p_j = e^{d_j} / s
//   ln p_j = d_j - ln s,   H = -sum p_j ln p_j = ln s - (sum e^{d_j} d_j) / s
// One pass keeps the running (m, s, w = sum e^d d); a new maximum m' rescales
//   s <- s f,  w <- (w + s (m - m')/T) f,  f = e^{(m - m')/T}.
// All sums, maxima and statistics are float32 whatever the logits' type.
#include <math.h>

#include "common.cuh"

namespace sffn {
namespace {

constexpr int TOP_MAX = 128;          // alternatives a row (and entries of a teacher's list)
constexpr float LOWEST = -3.402823466e38f;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
// Exponents below this give e^d = 0 in float32; the clamp keeps 0 * -inf out of w.
constexpr float D_MIN = -200.0f;

// Rows of a [rows / inner, inner, V] tensor whose last dimension is dense.
struct RowMap {
    int64_t inner, s_outer, s_inner;  // strides in elements
    __device__ __forceinline__ int64_t at(int64_t r) const { return (r / inner) * s_outer + (r % inner) * s_inner; }
};

template <int DT> struct Row {
    using bits = typename Elt<DT>::bits;
    static constexpr int N = 16 / sizeof(bits);  // elements of a 16-byte vector
};

// NaN-propagating max: a NaN logit has to reach s.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

template <int DT>
__device__ __forceinline__ void unpack(const uint4& q, float* x) {
    const uint32_t u[4] = {q.x, q.y, q.z, q.w};
    if constexpr (DT == SFFN_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(u[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = Elt<DT>::to_f((uint16_t)u[i]);
            x[2 * i + 1] = Elt<DT>::to_f((uint16_t)(u[i] >> 16));
        }
    }
}

template <int DT>
__device__ __forceinline__ uint4 pack(const float* x) {
    uint32_t u[4];
    if constexpr (DT == SFFN_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = __float_as_uint(x[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            u[i] = (uint32_t)Elt<DT>::from_f(x[2 * i]) | ((uint32_t)Elt<DT>::from_f(x[2 * i + 1]) << 16);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
}

template <int DT>
__device__ __forceinline__ float load1(const void* p, int64_t i) {
    return Elt<DT>::to_f(reinterpret_cast<const typename Elt<DT>::bits*>(p)[i]);
}
__device__ __forceinline__ float load_code(const void* p, int64_t i, int code) {
    return code == SFFN_F32 ? load1<SFFN_F32>(p, i) : code == SFFN_BF16 ? load1<SFFN_BF16>(p, i) : load1<SFFN_F16>(p, i);
}
__device__ __forceinline__ int64_t load_index(const void* p, int64_t i, int bytes) {
    return bytes == 8 ? reinterpret_cast<const int64_t*>(p)[i] : (int64_t) reinterpret_cast<const int32_t*>(p)[i];
}

// Where a row's 16-byte vectors begin: `head` single elements, `nvec` vectors, `tail` singles.
template <int DT>
struct Cut {
    int head, nvec, tail;
    __device__ __forceinline__ Cut(const void* row, int n) {
        constexpr int N = Row<DT>::N;
        const int es = 16 / N;
        const int mis = (int)(reinterpret_cast<uintptr_t>(row) & 15u) / es;
        head = min(n, mis ? N - mis : 0);
        nvec = (n - head) / N;
        tail = n - head - nvec * N;
    }
};

// The running (m, s, w) of one thread, exponents in units of log 2: c = log2(e) / T.
struct Soft {
    float m = LOWEST, s = 0.f, w = 0.f;
    __device__ __forceinline__ void raise(float to, float c) {
        const float by = fmaxf((m - to) * c, D_MIN);
        const float f = ex2(by);
        w = fmaf(s, by, w) * f;
        s *= f;
        m = to;
    }
    __device__ __forceinline__ void add(float x, float c) {
        const float d = max_nan((x - m) * c, D_MIN);
        const float e = ex2(d);
        s += e;
        w = fmaf(e, d, w);
    }
    __device__ __forceinline__ void one(float x, float c) {
        if (x > m) raise(x, c);
        add(x, c);
    }
};

// Sum over the block; every thread gets it.  `slots` holds a float per warp.
template <int NT>
__device__ __forceinline__ float block_sum(float v, float* slots) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
    __syncthreads();
    float r = 0.f;
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) r += slots[i];
    return r;
}
template <int NT>
__device__ __forceinline__ float block_max(float v, float* slots) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(FULL, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
    __syncthreads();
    float r = slots[0];
#pragma unroll
    for (int i = 1; i < NT / 32; ++i) r = fmaxf(r, slots[i]);
    return r;
}

// Joins the threads' running sums: afterwards every thread holds the row's.
template <int NT>
__device__ __forceinline__ void join(Soft& a, float c, float* slots) {
    const float m = block_max<NT>(a.m, slots);
    a.raise(m, c);
    a.s = block_sum<NT>(a.s, slots);
    a.w = block_sum<NT>(a.w, slots);
}

// Order of the alternatives: larger logits first, equal ones by lower index,
// NaN above all (as torch.sort has it); -0 equals +0.
__device__ __forceinline__ uint32_t order_bits(float x) {
    if (x != x) return 0xFFFFFFFFu;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float order_value(uint32_t o) {
    return __uint_as_float((o & 0x80000000u) ? o & 0x7FFFFFFFu : ~o);
}
__device__ __forceinline__ unsigned long long order_key(float x, int i) {
    return ((unsigned long long)order_bits(x) << 32) | (0xFFFFFFFFu - (uint32_t)i);
}

// f(x, index) for every element of the row that this thread owns.
template <int DT, int NT, class F>
__device__ __forceinline__ void each(const void* row, const Cut<DT>& cut, F&& f) {
    constexpr int N = Row<DT>::N;
    const int t = threadIdx.x;
    if (t < cut.head) f(load1<DT>(row, t), t);
    const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<const typename Elt<DT>::bits*>(row) + cut.head);
    for (int v = t; v < cut.nvec; v += NT) {
        float x[N];
        unpack<DT>(__ldg(q + v), x);
#pragma unroll
        for (int j = 0; j < N; ++j) f(x[j], cut.head + v * N + j);
    }
    const int at = cut.head + cut.nvec * N + t;
    if (t < cut.tail) f(load1<DT>(row, at), at);
}

// ---------------------------------------------------------------------------
// Log probabilities, entropy and top alternatives
// ---------------------------------------------------------------------------
struct ScoreArgs {
    const void* logits;
    RowMap map;
    int64_t rows;
    int vocab;
    const void* targets;  // null: none
    int target_bytes;
    int64_t ignore;
    int top_k;
    float inv_t;
    float *logp, *entropy, *stats;
    int64_t* top_ids;
    float* top_logp;
    uint32_t* status;
};

template <int DT, int NT>
__global__ void __launch_bounds__(NT) score_kernel(const ScoreArgs a) {
    __shared__ float slots[NT / 32];
    __shared__ unsigned long long keys[TOP_MAX];
    __shared__ int hist[256];
    __shared__ unsigned long long prefix_s;
    __shared__ int need_s, count_s;
    const int t = threadIdx.x;
    const int64_t r = blockIdx.x;
    int64_t target = -1;
    if (a.targets) {
        target = load_index(a.targets, r, a.target_bytes);
        if (target == a.ignore) {  // the row is left out: nothing of it is read
            if (t == 0) {
                a.logp[r] = 0.f;
                a.entropy[r] = 0.f;
                a.stats[2 * r] = 0.f;
                a.stats[2 * r + 1] = 0.f;
            }
            for (int i = t; i < a.top_k; i += NT) {
                a.top_ids[r * a.top_k + i] = -1;
                a.top_logp[r * a.top_k + i] = -INFINITY;
            }
            return;
        }
    }
    const void* row = reinterpret_cast<const typename Elt<DT>::bits*>(a.logits) + a.map.at(r);
    const Cut<DT> cut(row, a.vocab);
    const float c = a.inv_t * LOG2E;
    Soft soft;
    each<DT, NT>(row, cut, [&](float x, int) { soft.one(x, c); });
    join<NT>(soft, c, slots);
    const float ln_s = soft.s > 0.f || soft.s != soft.s ? logf(soft.s) : -INFINITY;
    if (t == 0) {
        if (a.targets) {
            float lp = NAN;
            if (target >= 0 && target < a.vocab)
                lp = soft.s == 0.f ? -INFINITY : (load1<DT>(row, target) - soft.m) * a.inv_t - ln_s;
            else
                atomicOr(a.status, SFFN_STATUS_BAD_INDEX);
            a.logp[r] = lp;
        }
        a.entropy[r] = soft.s == 0.f ? 0.f : ln_s - soft.w / soft.s * LN2;
        a.stats[2 * r] = soft.m;
        a.stats[2 * r + 1] = soft.s;
    }
    if (a.top_k == 0) return;
    // The top_k-th largest key, eight bits at a time.
    if (t == 0) {
        prefix_s = 0;
        need_s = a.top_k;
        count_s = 0;
    }
    for (int shift = 56; shift >= 0; shift -= 8) {
        for (int i = t; i < 256; i += NT) hist[i] = 0;
        __syncthreads();
        const unsigned long long prefix = prefix_s;
        each<DT, NT>(row, cut, [&](float x, int i) {
            const unsigned long long k = order_key(x, i);
            if (shift == 56 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1);
        });
        __syncthreads();
        if (t == 0) {
            int need = need_s, b = 255;
            for (; b > 0 && hist[b] < need; --b) need -= hist[b];
            need_s = need;
            prefix_s = prefix | ((unsigned long long)b << shift);
        }
        __syncthreads();
    }
    const unsigned long long least = prefix_s;
    each<DT, NT>(row, cut, [&](float x, int i) {
        const unsigned long long k = order_key(x, i);
        if (k >= least) {
            const int at = atomicAdd(&count_s, 1);
            if (at < TOP_MAX) keys[at] = k;
        }
    });
    __syncthreads();
    for (int i = t; i < a.top_k; i += NT) {
        const unsigned long long k = keys[i];
        int rank = 0;
        for (int j = 0; j < a.top_k; ++j) rank += keys[j] > k;
        const float x = order_value((uint32_t)(k >> 32));
        a.top_ids[r * a.top_k + rank] = 0xFFFFFFFFu - (uint32_t)k;
        a.top_logp[r * a.top_k + rank] = soft.s == 0.f ? -INFINITY : (x - soft.m) * a.inv_t - ln_s;
    }
}

struct ScoreBwdArgs {
    const void* logits;
    RowMap map;
    int64_t rows;
    int vocab;
    const void* targets;
    int target_bytes;
    int64_t ignore;
    int top_k;
    float inv_t;
    const float *entropy, *stats;
    const int64_t* top_ids;
    const float *g_logp, *g_entropy, *g_top;  // null: zero
    void* grad;
    int64_t grad_ld;
    int per;  // elements of a row that one block writes
};

// Writes f(x_j, j) to grad for the block's share of the row; 16-byte stores
// where the gradient's row is aligned as the logits' is.
template <int DT, int NT, class F>
__device__ __forceinline__ void map_row(const void* row, void* out, int n, F&& f) {
    using bits = typename Elt<DT>::bits;
    constexpr int N = Row<DT>::N;
    const int t = threadIdx.x;
    const bits* src = reinterpret_cast<const bits*>(row);
    bits* dst = reinterpret_cast<bits*>(out);
    if (((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15u) != 0) {
        for (int i = t; i < n; i += NT) dst[i] = Elt<DT>::from_f(f(Elt<DT>::to_f(src[i])));
        return;
    }
    const Cut<DT> cut(row, n);
    if (t < cut.head) dst[t] = Elt<DT>::from_f(f(Elt<DT>::to_f(src[t])));
    const uint4* q = reinterpret_cast<const uint4*>(src + cut.head);
    uint4* o = reinterpret_cast<uint4*>(dst + cut.head);
    for (int v = t; v < cut.nvec; v += NT) {
        float x[N];
        unpack<DT>(__ldg(q + v), x);
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = f(x[j]);
        o[v] = pack<DT>(x);
    }
    const int at = cut.head + cut.nvec * N + t;
    if (t < cut.tail) dst[at] = Elt<DT>::from_f(f(Elt<DT>::to_f(src[at])));
}

template <int NT>
__device__ __forceinline__ void zero_row(void* out, int64_t bytes) {
    unsigned char* p = reinterpret_cast<unsigned char*>(out);
    const int64_t head = min(bytes, (int64_t)((16 - (reinterpret_cast<uintptr_t>(p) & 15u)) & 15u));
    const int64_t nv = (bytes - head) / 16;
    for (int64_t i = threadIdx.x; i < head; i += NT) p[i] = 0;
    for (int64_t i = threadIdx.x; i < nv; i += NT) reinterpret_cast<uint4*>(p + head)[i] = make_uint4(0, 0, 0, 0);
    for (int64_t i = head + nv * 16 + threadIdx.x; i < bytes; i += NT) p[i] = 0;
}

// e^d / s of one logit, and ln of it (clamped, so that 0 * ln 0 is 0).
struct Prob {
    float m, inv_t, inv_s, ln_s;
    __device__ __forceinline__ float p(float x) const { return expf((x - m) * inv_t) * inv_s; }
    __device__ __forceinline__ float ln(float x) const { return max_nan((x - m) * inv_t - ln_s, D_MIN); }
};

template <int DT, int NT>
__global__ void __launch_bounds__(NT) score_bwd_kernel(const ScoreBwdArgs a) {
    using bits = typename Elt<DT>::bits;
    const int t = threadIdx.x;
    const int64_t r = blockIdx.x;
    const int begin = blockIdx.y * a.per, n = min(a.per, a.vocab - begin);
    const bits* row = reinterpret_cast<const bits*>(a.logits) + a.map.at(r);
    bits* out = reinterpret_cast<bits*>(a.grad) + r * a.grad_ld;
    int64_t target = a.targets ? load_index(a.targets, r, a.target_bytes) : -1;
    const float s = a.stats[2 * r + 1];
    if (s == 0.f || (a.targets && target == a.ignore)) {
        zero_row<NT>(out + begin, (int64_t)n * sizeof(bits));
        return;
    }
    const bool has_target = target >= 0 && target < a.vocab;
    const float g = a.g_logp && has_target ? a.g_logp[r] : 0.f;
    const float gh = a.g_entropy ? a.g_entropy[r] : 0.f;
    const float* gt = a.g_top ? a.g_top + r * a.top_k : nullptr;
    float total = 0.f;
    if (gt) {  // every warp sums the row's top_k upstream gradients for itself
        for (int i = t & 31; i < a.top_k; i += 32) total += gt[i];
#pragma unroll
        for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(FULL, total, o);
    }
    const Prob pr{a.stats[2 * r], a.inv_t, 1.0f / s, logf(s)};
    const float base = -(total + g) - gh * a.entropy[r];
    auto f = [&](float x) { return a.inv_t * (pr.p(x) * (base - gh * pr.ln(x))); };
    map_row<DT, NT>(row + begin, out + begin, n, f);
    // The places with a gradient of their own, rewritten whole: the target and the alternatives.
    bool hit = false;
    __syncthreads();
    if (gt && t < a.top_k) {
        const int64_t id = a.top_ids[r * a.top_k + t];
        hit = id == target;
        if (id >= begin && id < begin + n)
            out[id] = Elt<DT>::from_f(f(Elt<DT>::to_f(row[id])) + a.inv_t * (gt[t] + (hit ? g : 0.f)));
    }
    if (!__syncthreads_or(hit) && t == 0 && has_target && target >= begin && target < begin + n)
        out[target] = Elt<DT>::from_f(f(Elt<DT>::to_f(row[target])) + a.inv_t * g);
}

// ---------------------------------------------------------------------------
// Distillation from a teacher's top log probabilities
// ---------------------------------------------------------------------------
// Entries (id_i, c_i) of a row: q_i = e^{c_i} / sum e^{c} (renorm) or e^{c_i}
// (bucket, where the rest q_r = 1 - sum q is one more class whose probability
// under the student is the mass off the list).  Loss and gradient:
//   L = sum q_i (ln q_i - ln p_{id_i}) [+ q_r (ln q_r - ln p_r)]
//   T dL/dx_j = p_j Q - sum_{i: id_i = j} q_i  on the list, Q = sum q [+ q_r]
//             = p_j (Q - q_r / p_r)            off it
// p_r = s_off / s with s_off summed over the classes off the list themselves:
// 1 - sum p_i would lose all digits where the list holds nearly everything.
struct DistillArgs {
    const void* logits;
    RowMap map;
    int64_t rows;
    int vocab;
    const void* ids;
    int id_bytes;
    const void* scores;
    int score_code;
    int k, bucket;
    float inv_t;
    float* loss;
    float* stats;  // [rows, 4]: m, s, the factor off the list, ln of renorm's sum or bucket's Q
    uint32_t* status;
};

// A listed mass this near to one leaves no rest: less is the scores' own rounding.
constexpr float REST_FLOOR = 1.0f / (1 << 20);

template <int DT, int NT>
__global__ void __launch_bounds__(NT) distill_kernel(const DistillArgs a) {
    using bits = typename Elt<DT>::bits;
    constexpr int N = Row<DT>::N;
    extern __shared__ uint32_t on_list[];  // bucket: a bit per class, shifted so that vectors start whole
    __shared__ float slots[NT / 32];
    __shared__ int ids[TOP_MAX];
    const int t = threadIdx.x;
    const int64_t r = blockIdx.x;
    const bits* row = reinterpret_cast<const bits*>(a.logits) + a.map.at(r);
    const Cut<DT> cut(row, a.vocab);
    const float c = a.inv_t * LOG2E;

    // The list: one entry a thread (threads past it hold none).
    int id = -1;
    float score = -INFINITY;
    if (t < a.k) {
        const int64_t j = load_index(a.ids, r * a.k + t, a.id_bytes);
        if (j >= 0 && j < a.vocab) {
            id = (int)j;
            score = load_code(a.scores, r * a.k + t, a.score_code);
        } else if (j != -1) {
            atomicOr(a.status, SFFN_STATUS_BAD_INDEX);
        }
        ids[t] = id;
    }
    const float top = block_max<NT>(score, slots);
    const float z = block_sum<NT>(id >= 0 && score != -INFINITY ? expf(score - (a.bucket ? 0.f : top)) : 0.f, slots);
    if (z == 0.f) {  // no entry of positive weight
        if (t == 0) {
            a.loss[r] = 0.f;
            for (int i = 0; i < 4; ++i) a.stats[4 * r + i] = 0.f;
        }
        return;
    }
    const float ln_z = a.bucket ? 0.f : top + logf(z);
    const float ln_q = score - ln_z;
    const float q = id >= 0 ? expf(ln_q) : 0.f;

    // bits of the classes on the list
    const int pad = (N - cut.head % N) % N;
    bool first = id >= 0, all_listed = false;
    if (a.bucket) {
        for (int i = t; i < (a.vocab + pad + 31) / 32; i += NT) on_list[i] = 0;
        __syncthreads();
        if (id >= 0) atomicOr(&on_list[(id + pad) >> 5], 1u << ((id + pad) & 31));
        for (int i = 0; i < t && i < a.k && first; ++i) first = ids[i] != id;
        all_listed = __syncthreads_count(first) == a.vocab;
    }
    Soft soft;
    each<DT, NT>(row, cut, [&](float x, int i) {
        if (a.bucket && ((on_list[(i + pad) >> 5] >> ((i + pad) & 31)) & 1)) return;
        soft.one(x, c);
    });
    join<NT>(soft, c, slots);
    const float x = id >= 0 ? Elt<DT>::to_f(row[id]) : 0.f;
    float m = soft.m, s = soft.s, off = 0.f;
    if (a.bucket) {
        m = block_max<NT>(id >= 0 ? fmaxf(x, soft.m) : soft.m, slots);
        off = soft.s * ex2(fmaxf((soft.m - m) * c, D_MIN));
        s = off + block_sum<NT>(first ? ex2(max_nan((x - m) * c, D_MIN)) : 0.f, slots);
    }
    const float ln_s = s == 0.f ? -INFINITY : logf(s);
    const float ln_p = s == 0.f ? -INFINITY : (x - m) * a.inv_t - ln_s;
    float loss = block_sum<NT>(q != 0.f ? q * (ln_q - ln_p) : 0.f, slots);
    if (t == 0) {
        float factor = 1.f, more = ln_z;
        if (a.bucket) {
            float rest = 1.f - z;
            if (rest < REST_FLOOR || all_listed) rest = 0.f;
            more = z + rest;
            factor = more;
            if (rest > 0.f) {
                loss += rest * (logf(rest) - (logf(off) - ln_s));
                if (off > 0.f) factor -= rest * s / off;
            }
        }
        a.loss[r] = loss;
        a.stats[4 * r] = m;
        a.stats[4 * r + 1] = s;
        a.stats[4 * r + 2] = factor;
        a.stats[4 * r + 3] = more;
    }
}

struct DistillBwdArgs {
    const void* logits;
    RowMap map;
    int64_t rows;
    int vocab;
    const void* ids;
    int id_bytes;
    const void* scores;
    int score_code;
    int k, bucket;
    float inv_t;
    const float *stats, *g_loss;
    void* grad;
    int64_t grad_ld;
    int per;
};

template <int DT, int NT>
__global__ void __launch_bounds__(NT) distill_bwd_kernel(const DistillBwdArgs a) {
    using bits = typename Elt<DT>::bits;
    __shared__ int ids[TOP_MAX];
    __shared__ float qs[TOP_MAX];
    const int t = threadIdx.x;
    const int64_t r = blockIdx.x;
    const int begin = blockIdx.y * a.per, n = min(a.per, a.vocab - begin);
    const bits* row = reinterpret_cast<const bits*>(a.logits) + a.map.at(r);
    bits* out = reinterpret_cast<bits*>(a.grad) + r * a.grad_ld;
    const float s = a.stats[4 * r + 1];
    if (s == 0.f) {
        zero_row<NT>(out + begin, (int64_t)n * sizeof(bits));
        return;
    }
    const float g = a.g_loss[r] * a.inv_t, factor = a.stats[4 * r + 2], more = a.stats[4 * r + 3];
    const float Q = a.bucket ? more : 1.f, ln_z = a.bucket ? 0.f : more;
    if (t < a.k) {
        const int64_t j = load_index(a.ids, r * a.k + t, a.id_bytes);
        const bool ok = j >= 0 && j < a.vocab;
        ids[t] = ok ? (int)j : -1;
        qs[t] = ok ? expf(load_code(a.scores, r * a.k + t, a.score_code) - ln_z) : 0.f;
    }
    const Prob pr{a.stats[4 * r], a.inv_t, 1.0f / s, 0.f};
    const float gf = g * factor;
    map_row<DT, NT>(row + begin, out + begin, n, [&](float x) { return pr.p(x) * gf; });
    __syncthreads();
    if (t < a.k) {
        const int id = ids[t];
        if (id >= begin && id < begin + n) {
            float q = 0.f;  // an id that stands twice has the sum of its weights, from either entry
            for (int i = 0; i < a.k; ++i) q += ids[i] == id ? qs[i] : 0.f;
            out[id] = Elt<DT>::from_f(g * (pr.p(Elt<DT>::to_f(row[id])) * Q - q));
        }
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
int check_logits(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t inner, int64_t s_outer,
                 int64_t s_inner, float inv_t) {
    if (!dtype_ok(dtype)) return SFFN_ERR_DTYPE;
    if (rows < 0 || vocab < 1 || inner < 1 || s_outer < 0 || s_inner < 0) return SFFN_ERR_ARG;
    if (!(inv_t > 0.f) || !isfinite(inv_t)) return SFFN_ERR_ARG;
    if (rows > 0 && !logits) return SFFN_ERR_ARG;
    if (rows > 0x7fffffffll || vocab > (1ll << 30)) return SFFN_ERR_TOO_LARGE;
    if (reinterpret_cast<uintptr_t>(logits) % esize_of(dtype)) return SFFN_ERR_ALIGN;
    return SFFN_OK;
}

// Elements of a row that one block of the backward writes: a whole number of
// 16-byte vectors of any type.
constexpr int BWD_THREADS = 256;
int64_t bwd_per(int64_t rows, int64_t vocab) {
    (void)rows;
    const int64_t per = 16384;
    return vocab < per ? vocab : per;
}

#define SFFN_BY_DTYPE(dtype, CALL)                                  \
    do {                                                            \
        if (dtype == SFFN_F32) { CALL(SFFN_F32); }                  \
        else if (dtype == SFFN_BF16) { CALL(SFFN_BF16); }           \
        else { CALL(SFFN_F16); }                                    \
    } while (0)

}  // namespace
}  // namespace sffn

using namespace sffn;

extern "C" int sffn_token_logprobs(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t inner,
                                   int64_t s_outer, int64_t s_inner, const void* targets, int target_bytes,
                                   int64_t ignore_index, int top_k, float inv_t, float* logp, float* entropy,
                                   float* stats, int64_t* top_ids, float* top_logp, uint32_t* status_dev,
                                   void* stream) {
    if (int rc = check_logits(logits, dtype, rows, vocab, inner, s_outer, s_inner, inv_t)) return rc;
    if (targets && target_bytes != 4 && target_bytes != 8) return SFFN_ERR_ARG;
    if (top_k < 0 || top_k > vocab) return SFFN_ERR_ARG;
    if (top_k > TOP_MAX) return SFFN_ERR_TOO_LARGE;
    if (rows == 0) return SFFN_OK;
    if (!entropy || !stats || !status_dev || (targets && !logp) || (top_k && (!top_ids || !top_logp)))
        return SFFN_ERR_ARG;
    SFFN_BIND(scope, logits);
    const ScoreArgs a{logits, {inner, s_outer, s_inner}, rows, (int)vocab, targets, target_bytes, ignore_index,
                      top_k, inv_t, logp, entropy, stats, top_ids, top_logp, status_dev};
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
#define SFFN_CALL(DT) score_kernel<DT, 512><<<(unsigned)rows, 512, 0, st>>>(a)
    SFFN_BY_DTYPE(dtype, SFFN_CALL);
#undef SFFN_CALL
    SFFN_CHECK_LAUNCH();
    return SFFN_OK;
}

extern "C" int sffn_token_logprobs_bwd(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t inner,
                                       int64_t s_outer, int64_t s_inner, const void* targets, int target_bytes,
                                       int64_t ignore_index, const int64_t* top_ids, int top_k, float inv_t,
                                       const float* stats, const float* entropy, const float* g_logp,
                                       const float* g_entropy, const float* g_top, void* grad, int64_t grad_ld,
                                       void* stream) {
    if (int rc = check_logits(logits, dtype, rows, vocab, inner, s_outer, s_inner, inv_t)) return rc;
    if (targets && target_bytes != 4 && target_bytes != 8) return SFFN_ERR_ARG;
    if (top_k < 0 || top_k > vocab || grad_ld < vocab) return SFFN_ERR_ARG;
    if (top_k > TOP_MAX) return SFFN_ERR_TOO_LARGE;
    if (rows == 0) return SFFN_OK;
    if (!stats || !entropy || !grad || (g_top && top_k && !top_ids)) return SFFN_ERR_ARG;
    if (reinterpret_cast<uintptr_t>(grad) % esize_of(dtype)) return SFFN_ERR_ALIGN;
    SFFN_BIND(scope, logits);
    const int64_t per = bwd_per(rows, vocab);
    const int64_t blocks = (vocab + per - 1) / per;
    if (blocks > 65535) return SFFN_ERR_TOO_LARGE;
    const ScoreBwdArgs a{logits, {inner, s_outer, s_inner}, rows, (int)vocab, targets, target_bytes, ignore_index,
                         top_k, inv_t, entropy, stats, top_ids, g_logp, g_entropy, top_k ? g_top : nullptr, grad,
                         grad_ld, (int)per};
    const dim3 grid((unsigned)rows, (unsigned)blocks);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
#define SFFN_CALL(DT) score_bwd_kernel<DT, BWD_THREADS><<<grid, BWD_THREADS, 0, st>>>(a)
    SFFN_BY_DTYPE(dtype, SFFN_CALL);
#undef SFFN_CALL
    SFFN_CHECK_LAUNCH();
    return SFFN_OK;
}

namespace {
int check_list(const void* ids, int id_bytes, const void* scores, int score_dtype, int k, int tail) {
    if (!dtype_ok(score_dtype)) return SFFN_ERR_DTYPE;
    if (id_bytes != 4 && id_bytes != 8) return SFFN_ERR_ARG;
    if (k < 1 || (tail != SFFN_TAIL_RENORM && tail != SFFN_TAIL_BUCKET)) return SFFN_ERR_ARG;
    if (k > TOP_MAX) return SFFN_ERR_TOO_LARGE;
    if (!ids || !scores) return SFFN_ERR_ARG;
    return SFFN_OK;
}
}  // namespace

extern "C" int sffn_distill_topk(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t inner,
                                 int64_t s_outer, int64_t s_inner, const void* ids, int id_bytes,
                                 const void* scores, int score_dtype, int k, int tail, float inv_t, float* loss,
                                 float* stats, uint32_t* status_dev, void* stream) {
    if (int rc = check_logits(logits, dtype, rows, vocab, inner, s_outer, s_inner, inv_t)) return rc;
    if (rows == 0) return SFFN_OK;
    if (int rc = check_list(ids, id_bytes, scores, score_dtype, k, tail)) return rc;
    if (!loss || !stats || !status_dev) return SFFN_ERR_ARG;
    const int bucket = tail == SFFN_TAIL_BUCKET;
    const size_t smem = bucket ? ((size_t)vocab + 8 + 31) / 32 * 4 : 0;
    if (smem > 200 * 1024) return SFFN_ERR_TOO_LARGE;
    SFFN_BIND(scope, logits);
    const DistillArgs a{logits, {inner, s_outer, s_inner}, rows, (int)vocab, ids, id_bytes, scores, score_dtype,
                        k, bucket, inv_t, loss, stats, status_dev};
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
#define SFFN_CALL(DT)                                                                                          \
    if (smem > 32 * 1024)                                                                                      \
        SFFN_CUDA_TRY(cudaFuncSetAttribute(distill_kernel<DT, 512>, cudaFuncAttributeMaxDynamicSharedMemorySize, \
                                           200 * 1024));                                                       \
    distill_kernel<DT, 512><<<(unsigned)rows, 512, smem, st>>>(a)
    SFFN_BY_DTYPE(dtype, SFFN_CALL);
#undef SFFN_CALL
    SFFN_CHECK_LAUNCH();
    return SFFN_OK;
}

extern "C" int sffn_distill_topk_bwd(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t inner,
                                     int64_t s_outer, int64_t s_inner, const void* ids, int id_bytes,
                                     const void* scores, int score_dtype, int k, int tail, float inv_t,
                                     const float* stats, const float* g_loss, void* grad, int64_t grad_ld,
                                     void* stream) {
    if (int rc = check_logits(logits, dtype, rows, vocab, inner, s_outer, s_inner, inv_t)) return rc;
    if (grad_ld < vocab) return SFFN_ERR_ARG;
    if (rows == 0) return SFFN_OK;
    if (int rc = check_list(ids, id_bytes, scores, score_dtype, k, tail)) return rc;
    if (!stats || !g_loss || !grad) return SFFN_ERR_ARG;
    if (reinterpret_cast<uintptr_t>(grad) % esize_of(dtype)) return SFFN_ERR_ALIGN;
    SFFN_BIND(scope, logits);
    const int64_t per = bwd_per(rows, vocab);
    const int64_t blocks = (vocab + per - 1) / per;
    if (blocks > 65535) return SFFN_ERR_TOO_LARGE;
    const DistillBwdArgs a{logits, {inner, s_outer, s_inner}, rows, (int)vocab, ids, id_bytes, scores, score_dtype,
                           k, tail == SFFN_TAIL_BUCKET, inv_t, stats, g_loss, grad, grad_ld, (int)per};
    const dim3 grid((unsigned)rows, (unsigned)blocks);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
#define SFFN_CALL(DT) distill_bwd_kernel<DT, BWD_THREADS><<<grid, BWD_THREADS, 0, st>>>(a)
    SFFN_BY_DTYPE(dtype, SFFN_CALL);
#undef SFFN_CALL
    SFFN_CHECK_LAUNCH();
    return SFFN_OK;
}
