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
#include <cooperative_groups.h>
#include <math.h>

#include <type_traits>

#include "common.cuh"

namespace sffn {
namespace {

constexpr int SMS = 148;
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

// A vector that is read once: it takes no room in L1.
__device__ __forceinline__ uint4 load_once(const uint4* p) {
    uint4 q;
    asm("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w) : "l"(p));
    return q;
}

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

// The part of a row that one block reads: `head` single elements, `nvec` 16-byte
// vectors from the row's vector `first` on, `tail` singles from `tail_at` on.
// With `of` blocks to the row its vectors are split evenly, the head goes to
// the first block and the tail to the last.
template <int DT>
struct Cut {
    int lead;  // elements of the row before its first vector
    int head, first, nvec, tail, tail_at;
    __device__ __forceinline__ Cut(const void* row, int n, int which = 0, int of = 1) {
        constexpr int N = Row<DT>::N;
        const int es = 16 / N;
        const int mis = (int)(reinterpret_cast<uintptr_t>(row) & 15u) / es;
        lead = min(n, mis ? N - mis : 0);
        const int all = (n - lead) / N;
        tail_at = lead + all * N;
        first = (int)((int64_t)all * which / of);
        nvec = (int)((int64_t)all * (which + 1) / of) - first;
        head = which == 0 ? lead : 0;
        tail = which == of - 1 ? n - tail_at : 0;
    }
    // Index of element 0 of this part's vector v.
    __device__ __forceinline__ int at(int v) const { return lead + (first + v) * Row<DT>::N; }
    __device__ __forceinline__ const uint4* vectors(const void* row) const {
        return reinterpret_cast<const uint4*>(reinterpret_cast<const typename Elt<DT>::bits*>(row) + lead) + first;
    }
    __device__ __forceinline__ int begin() const { return head ? 0 : at(0); }
    __device__ __forceinline__ int end() const { return tail ? tail_at + tail : at(nvec); }
};

// Two float32 in one 64-bit register: sm_100a adds, multiplies and fuses both
// in one instruction, and the streaming loop is as near to the issue rate as
// to memory.
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t p, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// The largest of the values that these lanes of a warp bring, NaN left out.
__device__ __forceinline__ float max_of_lanes(unsigned lanes, float x) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "r"(lanes));
    return r;
}

// The running (m, s, w) of one thread, exponents in units of log 2: c = log2(e) / T.
// s and w are kept as pairs (even and odd elements).  m is an element of the row and
// none of the thread's own lies above it.  So a row's peak counts exactly 1 in s and
// 0 in w, a peaked row's small terms keep their digits, and s >= 1, ln p <= 0, H >= 0.
// (With m up to 2^32 behind, ln s and w / s came near 20 and their difference H lost
// five digits where it was 0.02.)  A warp's lanes raise m together, to the largest of
// their 32 vectors: about ln n times in n vectors of a lane, where lanes that raised
// each for itself would hold the warp up at most vectors.
// Without W (distillation, which wants no entropy) no w is kept, nor are exponents
// held above -inf for it (16384x50304 bf16 with the bucket: 8% of its time).
template <bool W>
struct Soft {
    float m = LOWEST;
    uint64_t s = 0, w = 0;
    __device__ __forceinline__ void raise(float to, float c) {
        const float by = fmaxf((m - to) * c, D_MIN);
        const float f = ex2(by);
        if (W) w = mul2(fma2(s, pair(by, by), w), pair(f, f));
        s = mul2(s, pair(f, f));
        m = to;
    }
    __device__ __forceinline__ void add(float x0, float x1, float c) {
        float d0, d1;
        unpair(mul2(add2(pair(x0, x1), pair(-m, -m)), pair(c, c)), d0, d1);
        if (W) {
            d0 = max_nan(d0, D_MIN);
            d1 = max_nan(d1, D_MIN);
        }
        const uint64_t e = pair(ex2(d0), ex2(d1));
        s = add2(s, e);
        if (W) w = fma2(e, pair(d0, d1), w);
    }
    // Before a vector whose largest element is `top`, by those `lanes` of a warp.
    __device__ __forceinline__ void reach(unsigned lanes, float top, float c) {
        if (__any_sync(lanes, top > m)) raise(fmaxf(m, max_of_lanes(lanes, top)), c);
    }
    __device__ __forceinline__ void one(float x, float c) {
        if (x > m) raise(x, c);
        add(x, -INFINITY, c);
    }
};

// Joins the threads' running sums: afterwards (m, s, w) is the block's, in every
// thread.  Two barriers; the slots are for this call alone.
template <int NT>
struct JoinSlots {
    float m[NT / 32];
    float2 sw[NT / 32];
};
template <int NT, bool W>
__device__ __forceinline__ void join(Soft<W>& a, float c, JoinSlots<NT>& slots, float& m, float& s, float& w) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    m = a.m;
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(FULL, m, o));
    if (lane == 0) slots.m[warp] = m;
    __syncthreads();
    m = slots.m[0];
#pragma unroll
    for (int i = 1; i < NT / 32; ++i) m = fmaxf(m, slots.m[i]);
    a.raise(m, c);
    float s1, w1;
    unpair(a.s, s, s1);
    unpair(a.w, w, w1);
    s += s1;
    w += w1;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        s += __shfl_xor_sync(FULL, s, o);
        w += __shfl_xor_sync(FULL, w, o);
    }
    if (lane == 0) slots.sw[warp] = make_float2(s, w);
    __syncthreads();
    s = w = 0.f;
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) {
        s += slots.sw[i].x;
        w += slots.sw[i].y;
    }
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

// f(x, index) for every element of the part that this thread owns.
template <int DT, int NT, class F>
__device__ __forceinline__ void each(const void* row, const Cut<DT>& cut, F&& f) {
    constexpr int N = Row<DT>::N;
    const int t = threadIdx.x;
    if (t < cut.head) f(load1<DT>(row, t), t);
    const uint4* q = cut.vectors(row);
    for (int v = t; v < cut.nvec; v += NT) {
        float x[N];
        unpack<DT>(__ldg(q + v), x);
#pragma unroll
        for (int j = 0; j < N; ++j) f(x[j], cut.at(v) + j);
    }
    if (t < cut.tail) f(load1<DT>(row, cut.tail_at + t), cut.tail_at + t);
}

// f(entry) for the k <= TOP_MAX entries of a row's list, dealt out to the block's threads.
template <int NT, class F>
__device__ __forceinline__ void entries(int k, F&& f) {
    if constexpr (NT >= TOP_MAX) {
        if ((int)threadIdx.x < k) f((int)threadIdx.x);
    } else {
        for (int e = threadIdx.x; e < k; e += NT) f(e);
    }
}

// One pass over the part: several vectors of a thread are loaded before the first
// is used: DEEP of them while a warp has as many (4 instead of 8: 16384x50304 bf16
// scored in 269 us instead of 251, distilled in 300 instead of 283), then AHEAD, and
// from the start beside the search of the alternatives, whose registers 8 would
// spill (8192 rows of it, k = 64: 257 us instead of 216).  A warp whose lanes have
// all of them runs without a check of each (with checks, and the lanes that pass
// them for each vector: 281 us and 314 with the bucket).  edit(x, index) may
// replace elements: a single one, and those of a vector where marks(places) has bit
// u set; seen(u, max, which) is told each vector's largest (u: its place among those;
// which: the vector, or -2 - index for a single element, with u = 0).  AGAIN: some
// are read again.
constexpr int AHEAD = 4, DEEP = 8;
template <int DT, int NT, bool AGAIN, bool W, class Marks, class Edit, class Seen>
__device__ __forceinline__ void stream(const void* row, const Cut<DT>& cut, float c, Soft<W>& soft, Marks&& marks, Edit&& edit,
                                       Seen&& seen) {
    constexpr int N = Row<DT>::N;
    const int t = threadIdx.x, lane = t & 31;
    auto single = [&](int i) {
        float x[1] = {load1<DT>(row, i)};
        edit(x, i, std::integral_constant<int, 1>());
        soft.one(x[0], c);
        seen(std::integral_constant<int, 0>(), x[0], -2 - i);
    };
    if (t < cut.head) single(t);
    const uint4* q = cut.vectors(row);
    int v0 = t, places = 0;  // before v0, of each thread
    // COUNT vectors of each thread.  WHOLE: all lanes of the warp have them all.
    auto go = [&](auto count, auto whole) {
        constexpr int COUNT = decltype(count)::value;
        constexpr bool WHOLE = decltype(whole)::value;
        uint4 raw[COUNT];
#pragma unroll
        for (int u = 0; u < COUNT; ++u)
            if (WHOLE || v0 + u * NT < cut.nvec) raw[u] = AGAIN ? __ldg(q + v0 + u * NT) : load_once(q + v0 + u * NT);
        const uint32_t marked = marks(places);
        auto use = [&](auto place) {
            constexpr int u = decltype(place)::value;
            const int v = v0 + u * NT;
            if (!WHOLE && v >= cut.nvec) return;
            float x[N];
            unpack<DT>(raw[u], x);
            if ((marked >> u) & 1) edit(x, cut.at(v), std::integral_constant<int, N>());
            float top = x[0];
#pragma unroll
            for (int j = 1; j < N; ++j) top = fmaxf(top, x[j]);
            const int with = WHOLE ? 32 : cut.nvec - (v - lane);  // lanes, the first ones, with a vector here
            soft.reach(with >= 32 ? FULL : (1u << with) - 1, top, c);
#pragma unroll
            for (int j = 0; j < N; j += 2) soft.add(x[j], x[j + 1], c);
            seen(place, top, v);
        };
        use(std::integral_constant<int, 0>());
        use(std::integral_constant<int, 1>());
        use(std::integral_constant<int, 2>());
        use(std::integral_constant<int, 3>());
        if constexpr (COUNT == DEEP) {
            use(std::integral_constant<int, 4>());
            use(std::integral_constant<int, 5>());
            use(std::integral_constant<int, 6>());
            use(std::integral_constant<int, 7>());
        }
        v0 += NT * COUNT;
        places += COUNT;
    };
    // (v0 - lane, by which a whole warp goes, is its first lane's)
    if constexpr (!AGAIN)
        while (v0 - lane + (DEEP - 1) * NT + 31 < cut.nvec) go(std::integral_constant<int, DEEP>(), std::true_type());
    while (v0 - lane + (AHEAD - 1) * NT + 31 < cut.nvec) go(std::integral_constant<int, AHEAD>(), std::true_type());
    while (v0 < cut.nvec) go(std::integral_constant<int, AHEAD>(), std::false_type());
    if (t < cut.tail) single(cut.tail_at + t);
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
    float *logp, *entropy, *stats;  // stats null: not kept
    int64_t* top_ids;
    float* top_logp;
    uint32_t* status;
    int parts;  // blocks to a row (a cluster)
};
constexpr int MAX_PARTS = 8;

// The alternatives of a block's part of a row as order keys, sorted, in `best`.
//
// The part falls into RUNS = 512 strided runs of vectors, and the threads bring
// the largest element of each: its order bits and its index, rounded up to its
// vector's last.  The k-th largest of these maxima is a lower bound of the k-th
// largest element above which little lies: 1.15 k elements of a shuffled row for
// k = 128.  One warp finds it, a bit of the order at a time; with many ties at
// the bound the index decides, also a bit at a time, so that a row of equal
// elements leaves about 8 k candidates.  Where a run's maximum reaches the bound
// the vector that holds it is read again, from L2, and all of the run where the
// largest of its other vectors (`second`) does too.  Where more than CAP elements
// reach it (the largest lie in few runs) or a NaN hides from the maxima, the k-th
// largest key is found exactly, eight bits a pass over the part.
constexpr int CAP = 1280;
constexpr int RUNS = 512;
struct TopSlots {
    unsigned long long keys[CAP];  // candidates
    unsigned long long best[TOP_MAX];
    uint32_t run_order[RUNS];
    int run_last[RUNS];
    int look[RUNS];  // read again: vectors from the front, runs from the back
    int hist[256];
    unsigned long long least;
    int vectors, runs, count, need, found;
};

// A value v with at least `need` of the warp's keys (PER a lane) >= v: the
// need-th largest key, from the highest bit in which the keys differ down, or a
// prefix of it that already parts `need` keys from the rest; 0 with fewer keys
// above 0.  Keys have LOW low bits that repeat the highest one, inverted.
template <int LOW, int PER>
__device__ __forceinline__ uint32_t kth_largest(const uint32_t (&key)[PER], int need) {
    uint32_t hi = 0, lo = 0xFFFFFFFFu;
    int some = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        hi = max(hi, key[i]);
        if (key[i]) {
            lo = min(lo, key[i]);
            ++some;
        }
    }
    if (__reduce_add_sync(FULL, some) < need) return 0;
    hi = __reduce_max_sync(FULL, hi);
    lo = __reduce_min_sync(FULL, lo);
    if (hi == lo) return hi;
    const int top = 31 - __clz(hi ^ lo);
    uint32_t v = top == 31 ? 0u : hi >> (top + 1) << (top + 1);
    for (int bit = top; bit >= LOW; --bit) {
        const uint32_t cand = v | (1u << bit);
        int n[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < PER; ++i) n[i & 3] += key[i] >= cand;
        const int all = __reduce_add_sync(FULL, (n[0] + n[1]) + (n[2] + n[3]));
        if (all >= need) v = cand;
        if (all == need) return v;
    }
    return v && !(v >> 31) ? v | ((1u << LOW) - 1) : v;
}
// Those bits of order_bits() of a type's values (finite or infinite).
template <int DT> constexpr int ORDER_LOW = DT == SFFN_F32 ? 0 : DT == SFFN_BF16 ? 16 : 13;
constexpr uint32_t ORDER_NEG_INF = 0x007FFFFFu;  // order_bits(-inf), the lowest

// A warp's 32 keys, one a lane, sorted: the largest in lane 0.
__device__ __forceinline__ unsigned long long sort_lanes(unsigned long long key) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int run = 2; run <= 32; run <<= 1)
#pragma unroll
        for (int step = run >> 1; step; step >>= 1) {
            const unsigned long long other = __shfl_xor_sync(FULL, key, step);
            const bool larger = ((lane & step) == 0) == ((lane & run) == 0);  // which of the two stays here
            if ((key < other) == larger) key = other;
        }
    return key;
}

// The k largest of z.keys[0 .. z.count), which are distinct, sorted into z.best;
// z.found of them.  A key's place is the number of larger ones.  Where several
// threads can share a key they count them one by one; with more keys the warps
// sort lists of 32 and look each key up in the other lists (8192x50304 bf16: k = 64
// 209 us, one by one 216; k = 128 244, one by one 286).
template <int NT>
__device__ __forceinline__ void sort_keys(int k, TopSlots& z) {
    const int t = threadIdx.x, lane = t & 31, count = z.count;
    int most = 0;
    auto place = [&](unsigned long long key, int above) {
        z.best[above] = key;
        most = max(most, above + 1);
    };
    if (count * 2 <= NT) {
        int lanes = 2;  // threads that share a key
        while (lanes < 32 && count * lanes * 2 <= NT) lanes *= 2;
        const int i = t / lanes;
        const unsigned long long key = i < count ? z.keys[i] : 0;
        int above = 0;
#pragma unroll 4
        for (int j = t % lanes; j < count; j += lanes) above += z.keys[j] > key;
        for (int o = 1; o < lanes; o <<= 1) above += __shfl_xor_sync(FULL, above, o);
        if (i < count && t % lanes == 0 && above < k) place(key, above);
    } else {
        static_assert(CAP % 32 == 0, "whole lists");
        const int lists = (count + 31) / 32;
        for (int l = t / 32; l < lists; l += NT / 32) {
            const int i = l * 32 + lane;
            z.keys[i] = sort_lanes(i < count ? z.keys[i] : 0);
        }
        __syncthreads();
        for (int l = t / 32; l < lists; l += NT / 32) {
            const unsigned long long key = z.keys[l * 32 + lane];
            int above = lane;
#pragma unroll 2
            for (int m = 0; m < lists; ++m) {
                if (m == l) continue;
                const unsigned long long* list = z.keys + m * 32;
                int larger = 0;
#pragma unroll
                for (int step = 16; step; step >>= 1) larger += list[larger + step - 1] > key ? step : 0;
                above += larger + (list[larger] > key);
            }
            if (key && above < k) place(key, above);
        }
    }
    most = __reduce_max_sync(FULL, most);
    if (lane == 0 && most) atomicMax(&z.found, most);
    __syncthreads();
}

// One warp's part of top_of: an order key that at least k elements reach, from the
// maxima of groups of GROUP runs.
template <int DT, int GROUP>
__device__ __forceinline__ unsigned long long bound_of(int k, const TopSlots& z) {
    constexpr int PER = RUNS / GROUP / 32;
    const int lane = threadIdx.x & 31;
    uint32_t order[PER], last[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        order[i] = 0;
        last[i] = 0xFFFFFFFFu;
#pragma unroll
        for (int g = 0; g < GROUP; ++g) {
            const int run = (g * PER + i) * 32 + lane;
            const uint32_t o = z.run_order[run], l = (uint32_t)z.run_last[run];
            last[i] = o > order[i] ? l : o == order[i] ? min(last[i], l) : last[i];
            order[i] = max(order[i], o);
        }
    }
    const uint32_t bound = kth_largest<ORDER_LOW<DT>>(order, k);
    int above = 0, equal = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        above += order[i] > bound;
        equal += order[i] == bound;
    }
    above = __reduce_add_sync(FULL, above);
    equal = __reduce_add_sync(FULL, equal);
    uint32_t place = 0;  // 2^32 - 1 - index from which an element at the bound counts
    if (bound && above < k && above + equal > 2 * k + 32) {
#pragma unroll
        for (int i = 0; i < PER; ++i) last[i] = order[i] == bound ? 0xFFFFFFFFu - last[i] : 0u;
        place = kth_largest<0>(last, k - above);
    }
    return ((unsigned long long)bound << 32) | place;
}

template <int DT, int NT>
__device__ __forceinline__ void top_of(const void* row, const Cut<DT>& cut, int k, const float (&top)[RUNS / NT],
                                       const float (&second)[RUNS / NT], const int (&held)[RUNS / NT], bool exact,
                                       TopSlots& z) {
    constexpr int N = Row<DT>::N, SUB = RUNS / NT;
    const int t = threadIdx.x;
    // Runs: NT > 128 has one a thread; NT = 128 one for each place u of AHEAD.
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
        z.run_order[u * NT + t] = held[u] != -1 ? order_bits(top[u]) : 0u;
        z.run_last[u * NT + t] = held[u] >= 0 ? cut.at(held[u]) + N - 1 : -2 - held[u];
    }
    if (t == 0) z.count = z.vectors = z.runs = z.found = 0;
    __syncthreads();
    if (t < 32 && !exact) {
        // few alternatives need few maxima: those of groups of four or two runs
        if (k <= RUNS / 16) z.least = bound_of<DT, 4>(k, z);
        else if (k <= RUNS / 8) z.least = bound_of<DT, 2>(k, z);
        else z.least = bound_of<DT, 1>(k, z);
    }
    __syncthreads();
    unsigned long long least = z.least;
    if (!exact) {
        const uint32_t bound = (uint32_t)(least >> 32), place = (uint32_t)least;
        const float floor = bound > ORDER_NEG_INF ? order_value(bound) : -INFINITY;
        auto reaches = [&](float x, int i) { return x > floor || (x == floor && 0xFFFFFFFFu - (uint32_t)i >= place); };
        auto single = [&](int i) {
            const float x = load1<DT>(row, i);
            if (!reaches(x, i)) return;
            const int to = atomicAdd(&z.count, 1);
            if (to < CAP) z.keys[to] = order_key(x, i);
        };
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
            const unsigned long long mine =
                ((unsigned long long)z.run_order[u * NT + t] << 32) | (0xFFFFFFFFu - (uint32_t)z.run_last[u * NT + t]);
            if (held[u] == -1 || mine < least) continue;
            if (second[u] >= floor) z.look[RUNS - 1 - atomicAdd(&z.runs, 1)] = u * NT + t;
            else if (held[u] >= 0) z.look[atomicAdd(&z.vectors, 1)] = held[u];
        }
        if (t < cut.head) single(t);
        if (t < cut.tail) single(cut.tail_at + t);
        __syncthreads();
        const uint4* q = cut.vectors(row);
        constexpr int STRIDE = SUB == 1 ? NT : NT * AHEAD;
        const int per = (cut.nvec + STRIDE - 1) / STRIDE, vectors = z.vectors, items = vectors + z.runs * per;
        for (int i0 = t; i0 < items; i0 += NT * AHEAD) {
            uint4 raw[AHEAD];
            int at[AHEAD];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int i = i0 + u * NT;
                at[u] = cut.nvec;
                if (i < vectors) {
                    at[u] = z.look[i];
                } else if (i < items) {
                    const int run = (i - vectors) / per;
                    at[u] = z.look[RUNS - 1 - run] + (i - vectors - run * per) * STRIDE;
                }
                if (at[u] < cut.nvec) raw[u] = __ldg(q + at[u]);
            }
            uint32_t hits = 0;  // bit u N + j: element j of vector u
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                if (at[u] >= cut.nvec) continue;
                float x[N];
                unpack<DT>(raw[u], x);
#pragma unroll
                for (int j = 0; j < N; ++j) hits |= (uint32_t)reaches(x[j], cut.at(at[u]) + j) << (u * N + j);
            }
            if (!hits) continue;
            int to = atomicAdd(&z.count, __popc(hits));
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                if (!((hits >> (u * N)) & ((1u << N) - 1))) continue;
                float x[N];
                unpack<DT>(raw[u], x);
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    if (!((hits >> (u * N + j)) & 1)) continue;
                    if (to < CAP) z.keys[to] = order_key(x[j], cut.at(at[u]) + j);
                    ++to;
                }
            }
        }
    }
    __syncthreads();
    if (exact || z.count > CAP) {
        __syncthreads();
        if (t == 0) {
            z.least = 0;
            z.need = k;
            z.count = 0;
        }
        for (int shift = 56; shift >= 0; shift -= 8) {
            for (int i = t; i < 256; i += NT) z.hist[i] = 0;
            __syncthreads();
            const unsigned long long prefix = z.least;
            each<DT, NT>(row, cut, [&](float x, int i) {
                const unsigned long long key = order_key(x, i);
                if (shift == 56 || (key >> (shift + 8)) == (prefix >> (shift + 8)))
                    atomicAdd(&z.hist[(key >> shift) & 255], 1);
            });
            __syncthreads();
            if (t == 0) {
                int need = z.need, b = 255;
                for (; b > 0 && z.hist[b] < need; --b) need -= z.hist[b];
                z.need = need;
                z.least = prefix | ((unsigned long long)b << shift);
            }
            __syncthreads();
        }
        least = z.least;
        each<DT, NT>(row, cut, [&](float x, int i) {
            const unsigned long long key = order_key(x, i);
            if (key >= least) {
                const int at = atomicAdd(&z.count, 1);
                if (at < CAP) z.keys[at] = key;
            }
        });
        __syncthreads();
    }
    sort_keys<NT>(k, z);
}

// What a block knows of its part of a row; the first block of a row's cluster
// joins its fellows' through distributed shared memory.
struct PartOut {
    float m, s, w;
};
__device__ __forceinline__ void join_parts(cooperative_groups::cluster_group& cluster, int of, PartOut& mine, float c,
                                           float& m, float& s, float& w) {
    PartOut all[MAX_PARTS];
#pragma unroll
    for (int i = 0; i < MAX_PARTS; ++i) {
        all[i] = {LOWEST, 0.f, 0.f};
        if (i < of) all[i] = *cluster.map_shared_rank(&mine, i);
        m = fmaxf(m, all[i].m);
    }
    s = w = 0.f;
#pragma unroll
    for (int i = 0; i < MAX_PARTS; ++i) {
        const float by = fmaxf((all[i].m - m) * c, D_MIN), f = ex2(by);
        s += all[i].s * f;
        w += fmaf(all[i].s, by, all[i].w) * f;
    }
}

// Blocks of NT threads that an SM holds: with 64 registers a thread, or 72 in small
// blocks, which spill nothing so.
constexpr int blocks_per_sm(int nt) { return nt < 128 ? 896 / nt : 1024 / nt; }

template <int DT, int NT, bool TOP>
__global__ void __launch_bounds__(NT, blocks_per_sm(NT)) score_kernel(const ScoreArgs a) {
    __shared__ JoinSlots<NT> slots;
    __shared__ PartOut mine;
    __shared__ typename std::conditional<TOP, TopSlots, int>::type top_slots;
    const int t = threadIdx.x;
    const int of = a.parts, which = of > 1 ? blockIdx.x % of : 0;
    const int64_t r = of > 1 ? blockIdx.x / of : blockIdx.x;
    int64_t target = -1;
    if (a.targets) {
        target = load_index(a.targets, r, a.target_bytes);
        if (target == a.ignore) {  // the row is left out: nothing of it is read
            if (which) return;
            if (t == 0) {
                a.logp[r] = 0.f;
                a.entropy[r] = 0.f;
                if (a.stats) a.stats[2 * r] = a.stats[2 * r + 1] = 0.f;
            }
            for (int i = t; i < a.top_k; i += NT) {
                a.top_ids[r * a.top_k + i] = -1;
                a.top_logp[r * a.top_k + i] = -INFINITY;
            }
            return;
        }
    }
    const void* row = reinterpret_cast<const typename Elt<DT>::bits*>(a.logits) + a.map.at(r);
    const Cut<DT> cut(row, a.vocab, which, of);
    const float c = a.inv_t * LOG2E;
    Soft<true> soft;
    constexpr int SUB = TOP ? RUNS / NT : 1;
    float top[SUB], second[SUB];  // of each run: the largest vector maximum, the largest of the other vectors'
    int held[SUB];                // the vector that holds it (-2 - index: a single element), -1 in an empty run
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
        top[u] = second[u] = -INFINITY;
        held[u] = u * NT + t < cut.nvec ? u * NT + t : -1;
    }
    stream<DT, NT, TOP>(row, cut, c, soft, [](int) { return 0u; }, [](float*, int, auto) {}, [&](auto place, float x, int which_vector) {
        if constexpr (TOP) {
            constexpr int u = SUB == 1 ? 0 : decltype(place)::value;
            second[u] = fmaxf(second[u], fminf(top[u], x));
            if (x > top[u]) {
                top[u] = x;
                held[u] = which_vector;
            }
        }
    });
    float m, s, w;
    join<NT>(soft, c, slots, m, s, w);
    if constexpr (TOP) top_of<DT, NT>(row, cut, a.top_k, top, second, held, s != s, top_slots);
    if (of > 1) {
        cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
        if (t == 0) mine = {m, s, w};
        cluster.sync();
        if (which == 0) join_parts(cluster, of, mine, c, m, s, w);
    }
    const float ln_s = s == 0.f ? -INFINITY : logf(s);
    if (which == 0 && t == 0) {
        if (a.targets) {
            float lp = NAN;
            if (target >= 0 && target < a.vocab)
                lp = s == 0.f ? -INFINITY : (load1<DT>(row, target) - m) * a.inv_t - ln_s;
            else
                atomicOr(a.status, SFFN_STATUS_BAD_INDEX);
            a.logp[r] = lp;
        }
        a.entropy[r] = s == 0.f ? 0.f : ln_s - w / s * LN2;
        if (a.stats) {
            a.stats[2 * r] = m;
            a.stats[2 * r + 1] = s;
        }
    }
    if constexpr (TOP) {
        auto put = [&](int i, unsigned long long key) {
            const float x = order_value((uint32_t)(key >> 32));
            a.top_ids[r * a.top_k + i] = 0xFFFFFFFFu - (uint32_t)key;
            a.top_logp[r * a.top_k + i] = s == 0.f ? -INFINITY : (x - m) * a.inv_t - ln_s;
        };
        if (of == 1) {
            for (int i = t; i < a.top_k; i += NT) put(i, top_slots.best[i]);
        } else if (which == 0) {
            // The parts' sorted lists: with the ceil(k / of)-th key of each at or above
            // the least of those, k keys are; only such keys are sorted again.
            cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
            const int k = a.top_k, deep = (k + of - 1) / of - 1;
            int* found = top_slots.look;  // of each part
            if (t == 0) top_slots.count = 0;
            if (t < of) found[t] = cluster.map_shared_rank(&top_slots, t)->found;
            __syncthreads();
            // every part's list of at most 128 keys, several keys a thread in flight
            constexpr int PER = MAX_PARTS * TOP_MAX / NT;
            unsigned long long key[PER], least = ~0ull;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int l = (i * NT + t) / TOP_MAX, j = (i * NT + t) % TOP_MAX;
                key[i] = l < of && j < found[l] ? cluster.map_shared_rank(&top_slots, l)->best[j] : 0;
                if (l < of && j == deep) top_slots.keys[l] = key[i];
            }
            __syncthreads();
            for (int l = 0; l < of; ++l) least = min(least, top_slots.keys[l]);
            __syncthreads();
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (key[i] && key[i] >= least) top_slots.keys[atomicAdd(&top_slots.count, 1)] = key[i];
            __syncthreads();
            sort_keys<NT>(k, top_slots);
            for (int i = t; i < k; i += NT) put(i, top_slots.best[i]);
        }
    }
    if (of > 1) cooperative_groups::this_cluster().sync();  // nobody leaves while the first block reads
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

// Writes f of the block's share of a row: f(x, n) replaces n elements in place.
// 16-byte accesses where the gradient's row is aligned as the logits' is.  FINAL:
// nothing of the row is read or written again, so its lines need no room in L1
// and may leave L2 at once (16384x50304 bf16 with blocks of 16384 elements: 568 us
// instead of 583; with places rewritten afterwards it would be 657 instead of 610).
template <int DT, int NT, bool FINAL, class F>
__device__ __forceinline__ void map_row(const void* row, void* out, int n, F&& f) {
    using bits = typename Elt<DT>::bits;
    constexpr int N = Row<DT>::N, AHEAD = 4;
    const int t = threadIdx.x;
    const bits* src = reinterpret_cast<const bits*>(row);
    bits* dst = reinterpret_cast<bits*>(out);
    auto single = [&](int i) {
        float x[2] = {Elt<DT>::to_f(src[i]), 0.f};
        f(x, std::integral_constant<int, 2>());
        dst[i] = Elt<DT>::from_f(x[0]);
    };
    if (((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15u) != 0) {
        for (int i = t; i < n; i += NT) single(i);
        return;
    }
    const Cut<DT> cut(row, n);
    if (t < cut.head) single(t);
    const uint4* q = reinterpret_cast<const uint4*>(src + cut.head);
    uint4* o = reinterpret_cast<uint4*>(dst + cut.head);
    for (int v0 = t; v0 < cut.nvec; v0 += NT * AHEAD) {
        uint4 raw[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
            if (v0 + u * NT < cut.nvec) raw[u] = FINAL ? load_once(q + v0 + u * NT) : __ldg(q + v0 + u * NT);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            if (v0 + u * NT >= cut.nvec) break;
            float x[N];
            unpack<DT>(raw[u], x);
            f(x, std::integral_constant<int, N>());
            if constexpr (FINAL) __stcs(o + v0 + u * NT, pack<DT>(x));
            else o[v0 + u * NT] = pack<DT>(x);
        }
    }
    if (t < cut.tail) single(cut.head + cut.nvec * N + t);
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

// x -> a p + b p ln p for pairs of logits.  For 16-bit gradients one exponential
// of (x - m) log2(e) / T - log2 s, within 2^-19 of p where p is above 2^-60; for
// float32 ones e^d by expf and 1 / s apart, which keeps p to the last bits.
template <int DT>
struct Weigh {
    float m, inv_t, inv_s, ln_s, c, l2s;
    __device__ __forceinline__ Weigh(float m_, float s, float inv_t_)
        : m(m_), inv_t(inv_t_), inv_s(1.0f / s), ln_s(logf(s)), c(inv_t_ * LOG2E), l2s(log2f(s)) {}
    template <int N, bool LN>
    __device__ __forceinline__ void apply(float* x, float a, float b) const {
#pragma unroll
        for (int j = 0; j < N; j += 2) {
            if constexpr (DT == SFFN_F32) {
#pragma unroll
                for (int i = j; i < j + 2; ++i) {
                    const float d = (x[i] - m) * inv_t, p = expf(d) * inv_s;
                    x[i] = p * (LN ? fmaf(b, max_nan(d - ln_s, D_MIN), a) : a);
                }
            } else {
                float d0, d1;
                unpair(fma2(add2(pair(x[j], x[j + 1]), pair(-m, -m)), pair(c, c), pair(-l2s, -l2s)), d0, d1);
                if (LN) {
                    d0 = max_nan(d0, D_MIN);
                    d1 = max_nan(d1, D_MIN);
                }
                uint64_t f = pair(a, a);
                if (LN) f = fma2(pair(d0, d1), pair(b * LN2, b * LN2), f);
                unpair(mul2(pair(ex2(d0), ex2(d1)), f), x[j], x[j + 1]);
            }
        }
    }
    // One logit's value, the same bits as in a vector.
    __device__ __forceinline__ float one(float x, float a, float b) const {
        float v[2] = {x, x};
        if (b == 0.f) apply<2, false>(v, a, b);
        else apply<2, true>(v, a, b);
        return v[0];
    }
    template <int NT, bool FINAL>
    __device__ __forceinline__ void row(const void* row, void* out, int n, float a, float b) const {
        if (b == 0.f)
            map_row<DT, NT, FINAL>(row, out, n, [&](float* x, auto k) { apply<decltype(k)::value, false>(x, a, b); });
        else
            map_row<DT, NT, FINAL>(row, out, n, [&](float* x, auto k) { apply<decltype(k)::value, true>(x, a, b); });
    }
};

// (with the 54 registers it would take unbounded: 539 us where it takes 509)
template <int DT, int NT>
__global__ void __launch_bounds__(NT, NT < 128 ? 32 : 1280 / NT) score_bwd_kernel(const ScoreBwdArgs a) {
    using bits = typename Elt<DT>::bits;
    const int t = threadIdx.x;
    const int64_t r = a.rows - 1 - blockIdx.x;  // the rows that the forward read last may still be in L2
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
    const Weigh<DT> weigh(a.stats[2 * r], s, a.inv_t);
    const float wa = -a.inv_t * (total + g + (gh != 0.f ? gh * a.entropy[r] : 0.f)), wb = -a.inv_t * gh;
    if (gt) weigh.template row<NT, false>(row + begin, out + begin, n, wa, wb);
    else weigh.template row<NT, true>(row + begin, out + begin, n, wa, wb);  // but for the target
    // The places with a gradient of their own, rewritten whole: the target and the alternatives.
    bool hit = false;
    __syncthreads();
    if (gt)
        entries<NT>(a.top_k, [&](int e) {
            const int64_t id = a.top_ids[r * a.top_k + e];
            hit |= id == target;
            if (id >= begin && id < begin + n)
                out[id] = Elt<DT>::from_f(weigh.one(Elt<DT>::to_f(row[id]), wa, wb) + a.inv_t * (gt[e] + (id == target ? g : 0.f)));
        });
    if (!__syncthreads_or(hit) && t == 0 && has_target && target >= begin && target < begin + n)
        out[target] = Elt<DT>::from_f(weigh.one(Elt<DT>::to_f(row[target]), wa, wb) + a.inv_t * g);
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
// The classes off the list are summed themselves, from their own maximum m_off:
//   ln p_r = (m_off - m) / T + ln s_off - ln s
// needs no p_r, which underflows where the list's logits stand far above the rest's
// (1 - sum p_i would lose all digits much sooner).  Such a row, with p_r below P_FAR,
// has its gradient off the list as q_off,j (p_r Q - q_r), where q_off,j = p_j / p_r =
// e^{(x_j - m_off) / T} / s_off.
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
    // [rows, 4]; all zero in a row without loss:
    //   renorm       m, s, the largest score, ln of the scores' sum from it
    //   bucket       m, s, the factor of p_j off the list, Q
    //   a far row    m_off, s_off, p_r - q_r, -s (Q is 1, and m the largest listed logit)
    float* stats;
    uint32_t* status;
    int parts;
};

// A listed mass this near to one leaves no rest: less is the scores' own rounding.
constexpr float REST_FLOOR = 1.0f / (1 << 20);
// From 2^-60 up p_j and q_r / p_r are within float32's range together.
constexpr float P_FAR = 1.0f / (1ll << 60);

template <int DT, int NT>
__global__ void __launch_bounds__(NT, blocks_per_sm(NT)) distill_kernel(const DistillArgs a) {
    using bits = typename Elt<DT>::bits;
    constexpr int N = Row<DT>::N;
    // bucket: a bit for each class of this block's part, and before them a bit for
    // each of its vectors, 32 of a thread's to a word
    extern __shared__ uint32_t marked_vectors[];
    __shared__ JoinSlots<NT> join_slots;
    __shared__ PartOut mine;
    __shared__ int ids[TOP_MAX];
    __shared__ float scores[TOP_MAX], logits_of[TOP_MAX];
    __shared__ bool firsts[TOP_MAX];
    const int t = threadIdx.x;
    const int of = a.parts, which = of > 1 ? blockIdx.x % of : 0;
    const int64_t r = of > 1 ? blockIdx.x / of : blockIdx.x;
    const bits* row = reinterpret_cast<const bits*>(a.logits) + a.map.at(r);
    const Cut<DT> cut(row, a.vocab, which, of);
    const float c = a.inv_t * LOG2E;

    // The list
    bool weighs = false;
    entries<NT>(a.k, [&](int e) {
        const int64_t j = load_index(a.ids, r * a.k + e, a.id_bytes);
        int id = -1;
        float score = -INFINITY, x = 0.f;
        if (j >= 0 && j < a.vocab) {
            id = (int)j;
            score = load_code(a.scores, r * a.k + e, a.score_code);
            x = Elt<DT>::to_f(row[id]);
        } else if (j != -1 && which == 0) {
            atomicOr(a.status, SFFN_STATUS_BAD_INDEX);
        }
        ids[e] = id;
        scores[e] = score;
        logits_of[e] = x;
        weighs |= score != -INFINITY;
    });
    // Classes are shifted so that a vector's bits lie in one word.
    const int pad = (N - cut.lead % N) % N;
    const int base = (cut.begin() + pad) & ~31;
    const int words = (cut.nvec + 32 * NT - 1) / (32 * NT) * NT;
    uint32_t* const on_list = marked_vectors + words;
    if (a.bucket)
        for (int i = t; i < words + (cut.end() + pad - base + 31) / 32; i += NT) marked_vectors[i] = 0;
    if (!__syncthreads_or(weighs)) {  // no entry of positive weight (every block of the row sees the same)
        if (t == 0 && which == 0) {
            a.loss[r] = 0.f;
            for (int i = 0; a.stats && i < 4; ++i) a.stats[4 * r + i] = 0.f;
        }
        return;
    }
    if (a.bucket) {
        bool twice = of > 1;  // an id that stands twice is one class: its first entry's
        entries<NT>(a.k, [&](int e) {
            const int id = ids[e];
            if (id < cut.begin() || id >= cut.end()) return;
            const int at = id + pad - base;
            twice |= (atomicOr(&on_list[at >> 5], 1u << (at & 31)) >> (at & 31)) & 1;
            const int v = (id - cut.at(0)) / N;
            if (id >= cut.at(0) && v < cut.nvec) atomicOr(&marked_vectors[v / (32 * NT) * NT + v % NT], 1u << (v / NT % 32));
        });
        twice = __syncthreads_or(twice);
        entries<NT>(a.k, [&](int e) {
            const int id = ids[e];
            bool first = id >= 0;
            if (twice)
#pragma unroll 8
                for (int i = 0; i < a.k; ++i) first &= !(i < e && ids[i] == id);
            firsts[e] = first;
        });
    }
    Soft<false> soft;
    static_assert(32 % DEEP == 0 && DEEP % AHEAD == 0, "the marks of vectors loaded together lie in one word");
    stream<DT, NT, false>(row, cut, c, soft,
                          [&](int places) { return a.bucket ? marked_vectors[places / 32 * NT + t] >> (places % 32) : 0u; },
                          [&](float* v, int i, auto count) {
                              if (!a.bucket) return;
                              constexpr int n = decltype(count)::value;
                              const uint32_t on = on_list[(i + pad - base) >> 5] >> ((i + pad - base) & 31);
#pragma unroll
                              for (int j = 0; j < n; ++j)
                                  if ((on >> j) & 1) v[j] = -INFINITY;
                          },
                          [](auto, float, int) {});
    float m, s, w;
    join<NT>(soft, c, join_slots, m, s, w);
    if (of > 1) {
        cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
        if (t == 0) mine = {m, s, w};
        cluster.sync();
        if (which == 0) join_parts(cluster, of, mine, c, m, s, w);
        cluster.sync();
        if (which) return;
    }

    // The rest is one warp's: the list's sums need no barrier so.
    if (t >= 32) return;
    constexpr int PER = TOP_MAX / 32;
    auto max_of = [](float v) {
#pragma unroll
        for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(FULL, v, o));
        return v;
    };
    auto sum_of = [](float v) {
#pragma unroll
        for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
        return v;
    };
    float score[PER], x[PER];
    bool on[PER];
    float top = -INFINITY, m_on = m;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = i * 32 + t;
        on[i] = e < a.k && ids[e] >= 0;
        score[i] = on[i] ? scores[e] : -INFINITY;
        x[i] = on[i] ? logits_of[e] : -INFINITY;
        top = fmaxf(top, score[i]);
        m_on = fmaxf(m_on, x[i]);
    }
    // q_i = e^{c_i - top} / z: the scores may be logits of any size, and top + ln z as one
    // number would cost q as many digits as top has before its point.
    float z = 0.f, rest = 0.f, ln_z = 0.f;
    if (a.bucket) {
        top = 0.f;
        // The rest is a difference of numbers near one and may be 2^-20 itself: the sum
        // and its terms take 64 bits (a float32 sum of 128 terms leaves 3% of a rest of 1e-5
        // in doubt).  32768x1024 bf16, k = 64: 3 us of 59.
        double listed = 0.0;
#pragma unroll 1
        for (int e = t; e < a.k; e += 32)
            if (ids[e] >= 0) listed += exp((double)scores[e]);
#pragma unroll
        for (int o = 16; o; o >>= 1) listed += __shfl_xor_sync(FULL, listed, o);
        z = (float)listed;
        rest = (float)(1.0 - listed);
    } else {
        top = max_of(top);
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (score[i] != -INFINITY) z += expf(score[i] - top);
        z = sum_of(z);
        ln_z = logf(z);
    }
    const float m_off = m, s_off = s;
    float off = 0.f;  // s_off from the row's maximum
    bool all_listed = false;
    if (a.bucket) {
        m = max_of(m_on);
        off = s_off * ex2(fmaxf((m_off - m) * c, D_MIN));
        float s_on = 0.f;
        int n = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (on[i] && firsts[i * 32 + t]) {
                s_on += ex2(max_nan((x[i] - m) * c, D_MIN));
                ++n;
            }
        s = off + sum_of(s_on);
        all_listed = __reduce_add_sync(FULL, n) == a.vocab;
    }
    const float ln_s = s == 0.f ? -INFINITY : logf(s);
    float loss = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const float ln_q = (score[i] - top) - ln_z, q = on[i] ? expf(ln_q) : 0.f;
        const float ln_p = s == 0.f ? -INFINITY : (x[i] - m) * a.inv_t - ln_s;
        if (q != 0.f) loss += q * (ln_q - ln_p);
    }
    loss = sum_of(loss);
    if (t == 0) {
        float factor = top, more = ln_z;
        if (a.bucket) {
            if (rest < REST_FLOOR || all_listed) rest = 0.f;
            more = z + rest;
            factor = more;
            if (rest > 0.f) {
                // One logarithm of q_r / p_r where that can be had: ln off and ln s are near ln V
                // each, and where the student is near the teacher their last bits are the loss.
                const bool far = s_off > 0.f && off < P_FAR * s;
                const float ln_ratio = far ? logf(rest) - ((m_off - m) * a.inv_t + logf(s_off) - ln_s)
                                           : s_off == 0.f ? INFINITY : logf(rest * (s / off));
                loss += rest * ln_ratio;
                if (far) {
                    factor = off / s - rest;
                    more = -s;
                    m = m_off;
                    s = s_off;
                } else if (off > 0.f) {
                    factor -= rest * s / off;
                }
            }
        }
        a.loss[r] = loss;
        if (!a.stats) return;
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
    const int64_t r = a.rows - 1 - blockIdx.x;  // the rows that the forward read last may still be in L2
    const int begin = blockIdx.y * a.per, n = min(a.per, a.vocab - begin);
    const bits* row = reinterpret_cast<const bits*>(a.logits) + a.map.at(r);
    bits* out = reinterpret_cast<bits*>(a.grad) + r * a.grad_ld;
    const float s = a.stats[4 * r + 1];
    if (s == 0.f) {
        zero_row<NT>(out + begin, (int64_t)n * sizeof(bits));
        return;
    }
    const float g = a.g_loss[r] * a.inv_t, third = a.stats[4 * r + 2], more = a.stats[4 * r + 3];
    const bool far = a.bucket && more < 0.f;
    const float Q = a.bucket && !far ? more : 1.f, factor = a.bucket ? third : 1.f;
    const float top = a.bucket ? 0.f : third, ln_z = a.bucket ? 0.f : more;
    entries<NT>(a.k, [&](int e) {
        const int64_t j = load_index(a.ids, r * a.k + e, a.id_bytes);
        const bool ok = j >= 0 && j < a.vocab;
        ids[e] = ok ? (int)j : -1;
        qs[e] = ok ? expf((load_code(a.scores, r * a.k + e, a.score_code) - top) - ln_z) : 0.f;
    });
    Weigh<DT> weigh(a.stats[4 * r], s, a.inv_t);
    weigh.template row<NT, false>(row + begin, out + begin, n, g * factor, 0.f);
    __syncthreads();
    if (far) {  // the listed places, whatever the reference off the list left there
        float m = a.stats[4 * r];
        for (int e = t & 31; e < a.k; e += 32)
            if (ids[e] >= 0) m = fmaxf(m, Elt<DT>::to_f(row[ids[e]]));
        weigh = Weigh<DT>(max_of_lanes(FULL, m), -more, a.inv_t);
    }
    entries<NT>(a.k, [&](int e) {
        const int id = ids[e];
        if (id < begin || id >= begin + n) return;
        float q = 0.f;  // an id that stands twice has the sum of its weights, from either entry
        for (int i = 0; i < a.k; ++i) q += ids[i] == id ? qs[i] : 0.f;
        out[id] = Elt<DT>::from_f(weigh.one(Elt<DT>::to_f(row[id]), g * Q, 0.f) - g * q);
    });
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
int check_logits(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t inner, int64_t s_outer,
                 int64_t s_inner, float inv_t) {
    if (!dtype_ok(dtype)) return SFFN_ERR_DTYPE;
    if (rows < 0 || vocab < 1 || inner < 1 || s_outer < 0 || s_inner < 0) return SFFN_ERR_ARG;
    if (!(inv_t > 0.f && inv_t < 2e30f)) return SFFN_ERR_ARG;  // D_MIN inv_t and c stay finite
    if (rows > 0 && !logits) return SFFN_ERR_ARG;
    if (rows > 0x7fffffffll || vocab > (1ll << 30)) return SFFN_ERR_TOO_LARGE;
    if (reinterpret_cast<uintptr_t>(logits) % esize_of(dtype)) return SFFN_ERR_ALIGN;
    return SFFN_OK;
}

// Elements of a row that one block of the backward writes (whole 16-byte vectors
// of any type): 65536, so that what a block does before its first vector counts
// little (16384x50304 bf16: 509 us, with 16384 elements 561; with a list 535 and
// 610); 16384 where that leaves fewer than 8192 blocks, whose last ones would
// run alone (1000x131072 float32: 172 us instead of 182); down to 4096 for a
// handful of rows (3x200003: 3.7 us, with 16384 elements 5.5).
int64_t bwd_per(int64_t rows, int64_t vocab) {
    int64_t per = 65536;
    const auto blocks = [&] { return rows * ((vocab + per - 1) / per); };
    while (per > 16384 && blocks() < 8192) per /= 2;
    while (per > 4096 && blocks() < 4 * SMS) per /= 2;
    return vocab < per ? vocab : per;
}
// By 256 threads, by 128 where that leaves a thread at most 8 vectors, by one warp
// where that does (rows of 4 KB: 32768x1024 bf16 score 28 us, by 128 threads 55;
// with a list 38 and 69): what a block does once a row counts most there.
int bwd_threads(int64_t per, int dtype) {
    const int64_t vectors = per * esize_of(dtype) / 16;
    return vectors <= 8 * 32 ? 32 : vectors <= 8 * 128 ? 128 : 256;
}

// How a forward row is shared out.  With more than eight rows an SM, one block
// takes a row: small blocks at different points of their rows keep memory busy
// where one large block would wait for its own end, and the smaller the block, the
// less a row costs beside its stream.  So it has `least` threads where the row is
// at most 32 KB or a thread's loads are one go, else `wide`.  Scores: 32 and 64
// (bf16, beside 128: 32768x1024 27 us and 71, 32768x8192 89 and 117; 16384x16640 94
// and 100, 2000x32000 27.2 and 28.3; from there on the two are even or 128 ahead:
// 16384x50304 250 and 249, 12000x32000 130 and 127, 4096x131072 170 and 167, float32
// 16384x16384 160 and 153).  Distillation with the bucket: 32 and 128 (32768x1024
// 59 us and 104, 32768x8192 143 and 174; 64 threads would gain nothing at 16384x50304,
// and at 131072 classes their bit lists leave room for few blocks: 226 us and 173).
// With alternatives: 128, for the runs.
// With fewer rows, a cluster of up to eight blocks of 128 takes a row, each a part
// of at least 2048 elements; where even those leave SMs half idle and a thread
// more than four vectors to read, the blocks have 512 threads.
struct Plan {
    int threads, parts;
};
Plan plan_rows(int64_t rows, int64_t vocab, int dtype, int least, int wide) {
    int parts = 1;
    while (parts < MAX_PARTS && rows * parts * 2 <= (int64_t)SMS * 8 && vocab / (parts * 2) >= 2048) parts *= 2;
    const int64_t vectors = vocab * esize_of(dtype) / 16 / parts;
    if (rows * parts <= 2 * SMS && vectors > 4 * 128) return {512, parts};
    if (parts > 1) return {128, parts};
    if (vectors <= DEEP * 32) return {least, 1};
    if (rows <= (int64_t)SMS * 8) return {128, 1};
    return {vectors <= 2048 ? least : wide, 1};
}

// Dynamic shared memory that distill_kernel may take: the bit lists of 1,400,000
// classes in one part come to 219,040 bytes, beside 2 KB of its own.  Calls set
// this one limit whatever they need themselves, since it is every host thread's:
// a smaller one could come between another thread's set and launch.
constexpr size_t DISTILL_SMEM = 220 * 1024;

// Launches kernel over rows x parts blocks, the parts of a row as a cluster.  Where the
// blocks of an SM could take more than 164 KB of shared memory (bit lists, 3 KB more a
// block), 164 KB are asked for: the rest is L1, where the loads in flight land.  With as
// many blocks as 228 KB hold, 1000x131072 float32 takes 102 us instead of 80, 1024x262144
// 217 instead of 180 (2048x262144 bf16, 205, takes 223); smaller lists need less than
// 164 KB and keep more L1 without (32768x8192 bf16 143 us, with 163).
template <class Args>
cudaError_t launch_rows(void (*kernel)(Args), const Plan& p, int64_t rows, size_t smem, cudaStream_t st, const Args& a) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * p.parts));
    cfg.blockDim = dim3((unsigned)p.threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    if (p.parts > 1) {
        at[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        at[cfg.numAttrs].val.clusterDim.x = (unsigned)p.parts;
        at[cfg.numAttrs].val.clusterDim.y = at[cfg.numAttrs].val.clusterDim.z = 1;
        ++cfg.numAttrs;
    }
    if (smem <= 128 * 1024 && (smem + 3 * 1024) * (blocks_per_sm(p.threads) + 1) > 164 * 1024) {
        at[cfg.numAttrs].id = cudaLaunchAttributePreferredSharedMemoryCarveout;
        at[cfg.numAttrs++].val.sharedMemCarveout = 72;  // per cent of 228 KB
    }
    cfg.attrs = at;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

// Whether pointers (or null) lie on their elements' boundaries.
bool lies(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

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
    if (!entropy || !status_dev || (targets && !logp) || (top_k && (!top_ids || !top_logp)))
        return SFFN_ERR_ARG;
    if ((targets && !lies(targets, target_bytes)) || !lies(logp, 4) || !lies(entropy, 4) || !lies(stats, 4) ||
        !lies(top_ids, 8) || !lies(top_logp, 4) || !lies(status_dev, 4))
        return SFFN_ERR_ALIGN;
    SFFN_BIND(scope, logits);
    const Plan p = plan_rows(rows, vocab, dtype, top_k ? 128 : 32, top_k ? 128 : 64);
    const ScoreArgs a{logits, {inner, s_outer, s_inner}, rows, (int)vocab, targets, target_bytes, ignore_index,
                      top_k, inv_t, logp, entropy, stats, top_ids, top_logp, status_dev, p.parts};
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
#define SFFN_CALL(DT)                                                                                    \
    SFFN_CUDA_TRY(launch_rows(top_k ? (p.threads == 512 ? score_kernel<DT, 512, true> : score_kernel<DT, 128, true>) \
                              : p.threads == 512 ? score_kernel<DT, 512, false>                          \
                              : p.threads == 128 ? score_kernel<DT, 128, false>                          \
                              : p.threads == 64 ? score_kernel<DT, 64, false> : score_kernel<DT, 32, false>, \
                              p, rows, 0, st, a))
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
    if (!lies(grad, esize_of(dtype)) || (targets && !lies(targets, target_bytes)) || !lies(top_ids, 8) || !lies(stats, 4) ||
        !lies(entropy, 4) || !lies(g_logp, 4) || !lies(g_entropy, 4) || !lies(g_top, 4))
        return SFFN_ERR_ALIGN;
    SFFN_BIND(scope, logits);
    const int64_t per = bwd_per(rows, vocab);
    const int64_t blocks = (vocab + per - 1) / per;
    if (blocks > 65535) return SFFN_ERR_TOO_LARGE;
    const ScoreBwdArgs a{logits, {inner, s_outer, s_inner}, rows, (int)vocab, targets, target_bytes, ignore_index,
                         top_k, inv_t, entropy, stats, top_ids, g_logp, g_entropy, top_k ? g_top : nullptr, grad,
                         grad_ld, (int)per};
    const dim3 grid((unsigned)rows, (unsigned)blocks);
    const int nt = bwd_threads(per, dtype);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
#define SFFN_CALL(DT)                                                                \
    if (nt == 32) score_bwd_kernel<DT, 32><<<grid, 32, 0, st>>>(a); \
    else if (nt == 128) score_bwd_kernel<DT, 128><<<grid, 128, 0, st>>>(a); \
    else score_bwd_kernel<DT, 256><<<grid, 256, 0, st>>>(a)
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
    if (!lies(ids, id_bytes) || !lies(scores, esize_of(score_dtype))) return SFFN_ERR_ALIGN;
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
    if (!loss || !status_dev) return SFFN_ERR_ARG;
    if (!lies(loss, 4) || !lies(stats, 4) || !lies(status_dev, 4)) return SFFN_ERR_ALIGN;
    const int bucket = tail == SFFN_TAIL_BUCKET;
    if (bucket && vocab > 1400000) return SFFN_ERR_TOO_LARGE;
    const Plan p = plan_rows(rows, vocab, dtype, 32, 128);
    // a bit for every class of a part (a vector more than its share, shifted by up
    // to 31 + 7 bits) and for every vector, in whole words of each thread
    const int64_t share = vocab / p.parts + 64;
    const size_t vectors = (share * esize_of(dtype) / 16 + 32 * p.threads) / (32 * p.threads) * p.threads;
    const size_t smem = bucket ? ((share + 31) / 32 + vectors) * 4 : 0;
    if (smem > DISTILL_SMEM) return SFFN_ERR_TOO_LARGE;
    SFFN_BIND(scope, logits);
    const DistillArgs a{logits, {inner, s_outer, s_inner}, rows, (int)vocab, ids, id_bytes, scores, score_dtype,
                        k, bucket, inv_t, loss, stats, status_dev, p.parts};
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
#define SFFN_CALL(DT)                                                                                    \
    auto* kernel = p.threads == 512 ? distill_kernel<DT, 512> : p.threads == 128 ? distill_kernel<DT, 128> \
                                                                 : distill_kernel<DT, 32>;             \
    if (smem > 32 * 1024)                                                                                \
        SFFN_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)DISTILL_SMEM)); \
    SFFN_CUDA_TRY(launch_rows(kernel, p, rows, smem, st, a))
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
    if (!lies(grad, esize_of(dtype)) || !lies(stats, 4) || !lies(g_loss, 4)) return SFFN_ERR_ALIGN;
    SFFN_BIND(scope, logits);
    const int64_t per = bwd_per(rows, vocab);
    const int64_t blocks = (vocab + per - 1) / per;
    if (blocks > 65535) return SFFN_ERR_TOO_LARGE;
    const DistillBwdArgs a{logits, {inner, s_outer, s_inner}, rows, (int)vocab, ids, id_bytes, scores, score_dtype,
                           k, tail == SFFN_TAIL_BUCKET, inv_t, stats, g_loss, grad, grad_ld, (int)per};
    const dim3 grid((unsigned)rows, (unsigned)blocks);
    const int nt = bwd_threads(per, dtype);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
#define SFFN_CALL(DT)                                                                  \
    if (nt == 32) distill_bwd_kernel<DT, 32><<<grid, 32, 0, st>>>(a); \
    else if (nt == 128) distill_bwd_kernel<DT, 128><<<grid, 128, 0, st>>>(a); \
    else distill_bwd_kernel<DT, 256><<<grid, 256, 0, st>>>(a)
    SFFN_BY_DTYPE(dtype, SFFN_CALL);
#undef SFFN_CALL
    SFFN_CHECK_LAUNCH();
    return SFFN_OK;
}
