// RMS norm after a block, gate, scaled residual add and the RMS norm before
// the next block, in one pass over the rows; forward and backward.
//
//   u  = y r1 w_post (post norm, r1 = rsqrt(mean y^2 + eps)) or y
//   x' = scale x + gate u
//   h  = x' r2 w_pre, r2 = rsqrt(mean x'^2 + eps)
// and, from dx' and dh, with xh = x' r2, yh = y r1, t = dh w_pre:
//   e   = dx' + r2 (t - xh mean(t xh))    dx = scale e
//   du  = gate e                          v  = du w_post
//   dy  = r1 (v - yh mean(v yh))          (post norm; dy = du without)
//   dw_pre = sum dh xh, dw_post = sum gate e yh, dgate = w_post sum e yh   (over the rows)
// With q = gate u, mean(v yh) = mean(q (dx' + r2 t)) - r2 mean(t xh) mean(q xh), so
// the backward adds up all it needs of a row at once and waits once a row.
// x' is recomputed from x and y, unrounded, for the bytes that reading it back
// would take.  All arithmetic, the row statistics and a block's sums over its rows are
// float32 (two to an instruction), the sums over the blocks 64 bits; each output is
// rounded once.
//
// Bound by memory: the forward moves four arrays of the stream's size, the
// backward six, and two things keep it from memory's rate: the instructions a
// row costs beside its arithmetic, and the waits for its sums.  So a thread keeps
// 8 columns for all its rows, with their weights and its sums of the weight
// gradients in registers, and works on up to 4 rows at a time (backward: one):
// their sums over a warp are formed together, each shuffle halving the number of
// values a lane still carries, with one barrier for all.  Meanwhile its own part
// of the next rows is copied to shared memory (cp.async; as each piece is copied
// and read by the same thread no barrier guards that ring).  Up to 16 warps share
// rows; rows wider than 4096 are split over a cluster of 2 or 4 blocks that
// exchange their sums through distributed shared memory.  The sums over rows are
// written once per block and joined by a second, small kernel in a fixed order:
// equal inputs give equal bits.
#include <cooperative_groups.h>
#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "sm100.cuh"

namespace sffn {
namespace {

namespace cg = cooperative_groups;

constexpr int CH = 8;          // columns of a thread
constexpr int MAX_WARPS = 16;  // warps of a block that share rows
constexpr int MAX_PARTS = 4;   // blocks (a cluster) that share rows
template <int DT> constexpr int BYTES = DT == SFFN_F32 ? 32 : 16;  // of a thread's columns
// Rows that a thread works on at a time, and stages of as many in its ring: what
// shared memory holds for 512 threads.
template <int TX, int TY, bool VEC> constexpr bool FWD_RING = VEC && BYTES<TX> + BYTES<TY> <= 48;
template <int TX, int TY, bool VEC> constexpr int FWD_ROWS = FWD_RING<TX, TY, VEC> ? 4 : 1;
template <int TX, int TY> constexpr int BWD_STAGES = BYTES<TX> + BYTES<TY> > 48 ? 3 : 4;
template <int TX, int TY> constexpr int STAGES = BYTES<TX> + BYTES<TY> == 48 ? 2 : 3;
// The backward's ring: float32 also where its rows are copied by single elements.
template <int TX, int TY, bool VEC> constexpr bool BWD_RING = VEC || (TX == SFFN_F32 && TY == SFFN_F32);
constexpr int SMS = 148;

__device__ __forceinline__ void store_code(void* p, int64_t i, int code, float v) {
    if (code == SFFN_F32) reinterpret_cast<float*>(p)[i] = v;
    else if (code == SFFN_BF16) reinterpret_cast<uint16_t*>(p)[i] = Elt<SFFN_BF16>::from_f(v);
    else reinterpret_cast<uint16_t*>(p)[i] = Elt<SFFN_F16>::from_f(v);
}

// Two float32 in one 64-bit register; sm_100a computes both in one instruction.
using Pair = uint64_t;
__device__ __forceinline__ Pair pair(float a, float b) {
    Pair r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ Pair both(float a) { return pair(a, a); }
__device__ __forceinline__ float2 unpair(Pair p) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
    return r;
}
__device__ __forceinline__ float sum_of(Pair p) {
    const float2 f = unpair(p);
    return f.x + f.y;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// A thread's eight columns, so that a warp's accesses are whole lines:
//   EIGHTS  eight neighbours (16-byte accesses of 16-bit types)
//   FOURS   four neighbours in each half of the warp's 256 (16-byte accesses of
//           float32, 8-byte ones of a 16-bit type beside it)
//   SINGLES every 32nd of the warp's 256 (rows that such accesses cannot reach)
enum { SINGLES = 0, FOURS = 1, EIGHTS = 2 };
constexpr int mode_of(int tx, int ty, bool vec) {
    return !vec ? SINGLES : tx == SFFN_F32 || ty == SFFN_F32 ? FOURS : EIGHTS;
}
template <int MODE>
struct Place {
    int from, width;  // the first column; the row's columns
    __device__ __forceinline__ Place(int warp, int lane, int start, int end)
        : from(start + warp * 32 * CH + lane * (MODE == EIGHTS ? 8 : MODE == FOURS ? 4 : 1)), width(end) {}
    __device__ __forceinline__ int col(int j) const { return from + j * 32; }  // SINGLES
    __device__ __forceinline__ bool full() const { return col(CH - 1) < width; }
};

// Two or four values as they lie in memory.
template <int DT>
__device__ __forceinline__ void unpack4(const uint4& q, Pair* x) {  // float32: four
    x[0] = pair(__uint_as_float(q.x), __uint_as_float(q.y));
    x[1] = pair(__uint_as_float(q.z), __uint_as_float(q.w));
}
template <int DT>
__device__ __forceinline__ Pair unpack2(uint32_t u) {
    return pair(Elt<DT>::to_f((uint16_t)u), Elt<DT>::to_f((uint16_t)(u >> 16)));
}

template <int DT, int MODE>
__device__ __forceinline__ void load8(const void* base, const Place<MODE>& pl, Pair* x) {
    using bits = typename Elt<DT>::bits;
    const bits* p = reinterpret_cast<const bits*>(base) + pl.from;
    if constexpr (MODE == EIGHTS) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = 0;
        if (pl.from < pl.width) {
            if constexpr (DT == SFFN_F32) {
                unpack4<DT>(reinterpret_cast<const uint4*>(p)[0], x);
                unpack4<DT>(reinterpret_cast<const uint4*>(p)[1], x + 2);
            } else {
                const uint4 q = *reinterpret_cast<const uint4*>(p);
                x[0] = unpack2<DT>(q.x);
                x[1] = unpack2<DT>(q.y);
                x[2] = unpack2<DT>(q.z);
                x[3] = unpack2<DT>(q.w);
            }
        }
    } else if constexpr (MODE == FOURS) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            x[2 * h] = x[2 * h + 1] = 0;
            if (pl.from + 128 * h < pl.width) {
                if constexpr (DT == SFFN_F32) {
                    unpack4<DT>(*reinterpret_cast<const uint4*>(p + 128 * h), x + 2 * h);
                } else {
                    const uint2 q = *reinterpret_cast<const uint2*>(p + 128 * h);
                    x[2 * h] = unpack2<DT>(q.x);
                    x[2 * h + 1] = unpack2<DT>(q.y);
                }
            }
        }
    } else if (pl.full()) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = pair(Elt<DT>::to_f(p[64 * i]), Elt<DT>::to_f(p[64 * i + 32]));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            x[i] = pair(pl.col(2 * i) < pl.width ? Elt<DT>::to_f(p[64 * i]) : 0.f,
                        pl.col(2 * i + 1) < pl.width ? Elt<DT>::to_f(p[64 * i + 32]) : 0.f);
    }
}

// The same of a weight or gate row, whose type is an argument; ones where there is none.
template <int MODE>
__device__ __forceinline__ void load_weight(const void* p, int code, int64_t offset, const Place<MODE>& pl, Pair* x) {
    if (!p) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = both(1.f);
    } else if (code == SFFN_F32) {
        load8<SFFN_F32, MODE>(reinterpret_cast<const float*>(p) + offset, pl, x);
    } else if (code == SFFN_BF16) {
        load8<SFFN_BF16, MODE>(reinterpret_cast<const uint16_t*>(p) + offset, pl, x);
    } else {
        load8<SFFN_F16, MODE>(reinterpret_cast<const uint16_t*>(p) + offset, pl, x);
    }
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float2 f) {
    uint32_t r;
    if constexpr (DT == SFFN_BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(f.y), "f"(f.x));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(f.y), "f"(f.x));
    return r;
}

template <int DT, int MODE>
__device__ __forceinline__ void store8(void* base, const Place<MODE>& pl, const Pair* x) {
    using bits = typename Elt<DT>::bits;
    bits* p = reinterpret_cast<bits*>(base) + pl.from;
    float2 f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = unpair(x[i]);
    if constexpr (MODE == EIGHTS) {
        if (pl.from >= pl.width) return;
        if constexpr (DT == SFFN_F32) {
            reinterpret_cast<float4*>(p)[0] = make_float4(f[0].x, f[0].y, f[1].x, f[1].y);
            reinterpret_cast<float4*>(p)[1] = make_float4(f[2].x, f[2].y, f[3].x, f[3].y);
        } else {
            *reinterpret_cast<uint4*>(p) = make_uint4(pack2<DT>(f[0]), pack2<DT>(f[1]), pack2<DT>(f[2]), pack2<DT>(f[3]));
        }
    } else if constexpr (MODE == FOURS) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (pl.from + 128 * h >= pl.width) continue;
            if constexpr (DT == SFFN_F32)
                *reinterpret_cast<float4*>(p + 128 * h) = make_float4(f[2 * h].x, f[2 * h].y, f[2 * h + 1].x, f[2 * h + 1].y);
            else
                *reinterpret_cast<uint2*>(p + 128 * h) = make_uint2(pack2<DT>(f[2 * h]), pack2<DT>(f[2 * h + 1]));
        }
    } else if (pl.full()) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            p[64 * i] = Elt<DT>::from_f(f[i].x);
            p[64 * i + 32] = Elt<DT>::from_f(f[i].y);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (pl.col(2 * i) < pl.width) p[64 * i] = Elt<DT>::from_f(f[i].x);
            if (pl.col(2 * i + 1) < pl.width) p[64 * i + 32] = Elt<DT>::from_f(f[i].y);
        }
    }
}

// gate x post weight of the gate row at `offset`
template <int MODE>
__device__ __forceinline__ void load_scale(const void* gate, int gate_code, int64_t offset, const void* post, int post_code,
                                           const Place<MODE>& pl, Pair* g) {
    Pair w[4];
    load_weight<MODE>(gate, gate_code, offset, pl, g);
    load_weight<MODE>(post, post_code, 0, pl, w);
#pragma unroll
    for (int i = 0; i < 4; ++i) g[i] = mul2(g[i], w[i]);
}

// A thread's own ring of rows: [stage][row][array][piece][thread].  A thread's
// part of a row is 1 piece of 16 bytes (EIGHTS), 2 of 16 (FOURS, float32) or 8
// bytes (FOURS, 16 bits), or 8 of 4 bytes (SINGLES, float32 alone; 16-bit
// elements of such rows come straight from global memory).
template <int DT, int MODE> constexpr int PIECES = MODE == EIGHTS ? 1 : MODE == FOURS ? 2 : 8;

__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory"); }

// `from`: the row's first column of this thread.
template <int DT, int MODE>
__device__ __forceinline__ void copy8(uint32_t to, int threads, const typename Elt<DT>::bits* from, const Place<MODE>& pl) {
    constexpr int N = PIECES<DT, MODE>, SIZE = BYTES<DT> / N;
    to += threadIdx.x * SIZE;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        constexpr int STEP = MODE == FOURS ? 128 : 32;  // columns from a piece to the next
        if (pl.from + STEP * i >= pl.width) continue;
        if constexpr (SIZE == 16)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + i * threads * SIZE), "l"(from + STEP * i) : "memory");
        else
            asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to + i * threads * SIZE), "l"(from + STEP * i), "n"(SIZE) : "memory");
    }
}
// Columns that no copy fills read as zero: clear8 at the start, for every stage.
template <int DT, int MODE>
__device__ __forceinline__ void clear8(uint32_t at, int threads) {
    constexpr int N = PIECES<DT, MODE>, SIZE = BYTES<DT> / N;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < SIZE; j += 4)
            asm volatile("st.shared.u32 [%0], %1;" ::"r"(at + (i * threads + threadIdx.x) * SIZE + j), "r"(0) : "memory");
}
template <int DT, int MODE>
__device__ __forceinline__ void take8(uint32_t from, int threads, Pair* x) {
    constexpr int N = PIECES<DT, MODE>, SIZE = BYTES<DT> / N;
    from += threadIdx.x * SIZE;
    if constexpr (SIZE == 16) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            uint4 q;
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w)
                         : "r"(from + i * threads * SIZE) : "memory");
            if constexpr (DT == SFFN_F32) {
                unpack4<DT>(q, x + 2 * i);
            } else {
                x[0] = unpack2<DT>(q.x);
                x[1] = unpack2<DT>(q.y);
                x[2] = unpack2<DT>(q.z);
                x[3] = unpack2<DT>(q.w);
            }
        }
    } else if constexpr (SIZE == 8) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            uint2 q;
            asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(q.x), "=r"(q.y) : "r"(from + i * threads * SIZE) : "memory");
            x[2 * i] = unpack2<DT>(q.x);
            x[2 * i + 1] = unpack2<DT>(q.y);
        }
    } else {
        float f[CH];
#pragma unroll
        for (int i = 0; i < CH; ++i)
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f[i % CH]) : "r"(from + i * threads * SIZE) : "memory");
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = pair(f[2 * i], f[2 * i + 1]);
    }
}

// Stores v at this block's shared address `to` in block `rank` of the cluster and
// counts its 4 bytes at that block's `barrier`.
__device__ __forceinline__ void send(uint32_t to, uint32_t barrier, int rank, float v) {
    asm volatile(
        "{\n\t.reg .b32 a, b;\n\t"
        "mapa.shared::cluster.u32 a, %0, %2;\n\t"
        "mapa.shared::cluster.u32 b, %1, %2;\n\t"
        "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b32 [a], %3, [b];\n\t}"
        ::"r"(to), "r"(barrier), "r"(rank), "r"(__float_as_uint(v)) : "memory");
}

// Sums of N values over the threads that share rows.  In a warp the lanes halve
// the values among them while they add: log2 N exchanges of N / 2, N / 4, ... values,
// then of one.  The warps' sums meet in slots, and every thread adds them up in
// the same order.  Two slot sets alternate: a set is written again only after the
// other set's barrier, which every reader of it has passed.
//
// In a cluster each warp stores its sums to every block's slots (st.async), and
// an mbarrier of each set counts the bytes: unlike the cluster's own barrier that
// does not wait until the rows' stores to global memory are acknowledged (float32
// 8192x8192 with bf16: 181 -> 155 us forward, 314 -> 273 us backward).  The wait
// acquires at the cluster's scope, since other blocks stored what it waits for, and is
// bounded: when it runs out it sets SFFN_STATUS_WAIT_TIMEOUT and no later one waits.
template <int N, bool WIDE, int SUBS>
struct RowSums {
    static constexpr int LANES = 32 / SUBS;
    static constexpr int POW = N <= 1 ? 1 : N <= 2 ? 2 : 4;
    static_assert(N <= 4, "one 16-byte slot a warp");
    float4* slots;  // [2][fold] of this group, zeroed
    int warps, warp, lane, bar, parts, part;
    int fold;  // the power of two that covers warps * parts
    uint64_t* filled;  // [2], of a cluster
    uint32_t* status;
    int set = 0;
    uint32_t phase = 0;  // bit i: the parity that set i's barrier completes next
    bool gave_up = false;
    __device__ __forceinline__ RowSums(float4* slots_, int fold_, int warps_, int warp_, int lane_, int bar_, int parts_, int part_,
                                       uint64_t* filled_, uint32_t* status_)
        : slots(slots_), warps(warps_), warp(warp_), lane(lane_), bar(bar_), parts(parts_), part(part_), fold(fold_),
          filled(filled_), status(status_) {}
    __device__ __forceinline__ void operator()(float (&v)[N]) {
        float w[POW];
#pragma unroll
        for (int i = 0; i < POW; ++i) w[i] = i < N ? v[i < N ? i : 0] : 0.f;
        int o = LANES / 2;
#pragma unroll
        for (int n = POW; n > 1; n >>= 1, o >>= 1) {
            const bool up = lane & o;
#pragma unroll
            for (int i = 0; i < n / 2; ++i) {
                const float keep = up ? w[i + n / 2] : w[i], give = up ? w[i] : w[i + n / 2];
                w[i] = keep + __shfl_xor_sync(FULL, give, o);
            }
        }
#pragma unroll
        for (; o; o >>= 1) w[0] += __shfl_xor_sync(FULL, w[0], o);
        if (SUBS > 1 || (!WIDE && fold == 1)) {  // one warp: value i is in lanes i * LANES / POW on
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = __shfl_sync(FULL, w[0], (SUBS > 1 ? lane & ~(LANES - 1) : 0) + i * (LANES / POW));
            return;
        }
        float4* s = slots + set;
        set ^= fold;
        float* mine = reinterpret_cast<float*>(s + part * warps + warp) + lane / (32 / POW);
        if constexpr (!WIDE) {
            if (lane % (32 / POW) == 0) *mine = w[0];
            asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(warps * 32) : "memory");
        } else {
            const int which = s != slots;
            uint64_t* full = filled + which;
            if (threadIdx.x == 0) mbar_arrive_expect_tx(full, parts * warps * POW * 4);
            if (lane % (32 / POW) == 0)
                for (int i = 0; i < parts; ++i) send(smem_u32(mine), smem_u32(full), i, w[0]);
            if (!gave_up && !mbar_wait_bounded<true>(full, (phase >> which) & 1)) {
                gave_up = true;
                atomicOr(status, SFFN_STATUS_WAIT_TIMEOUT);
            }
            phase ^= 1u << which;
        }
        float4 q = s[lane & (fold - 1)];
        if (WIDE && fold > 32) {
            const float4 p = s[(lane & (fold - 1)) + 32];
            q.x += p.x;
            q.y += p.y;
            q.z += p.z;
            q.w += p.w;
        }
        const float f[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = f[i];
        for (int d = min(fold, 32) >> 1; d; d >>= 1)
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(FULL, v[i], d);
    }
};
__device__ __forceinline__ int fold_of(int n) { return n <= 1 ? 1 : 1 << (32 - __clz(n - 1)); }
// Slots of a block: two sets of the fold of the warps for each group (at most
// 2 * MAX_WARPS in all), or of a cluster's warps.
constexpr int SLOTS = 2 * (MAX_PARTS * MAX_WARPS > 2 * MAX_WARPS ? MAX_PARTS * MAX_WARPS : 2 * MAX_WARPS);

// How rows lie on the threads of a launch.
struct Shape {
    int parts, cols;    // blocks to a row, columns of each but the last
    int warps, groups;  // warps of a block to a row, groups of them
    int64_t blocks;     // of the launch; a multiple of parts
    int64_t per;        // consecutive rows of one group
    __host__ __device__ int threads() const { return warps * groups * 32; }
    __host__ __device__ int64_t units() const { return blocks / parts * groups; }
};

struct NormArgs {
    const void *x, *y;  // y null: no block output, h = norm of x alone
    int64_t x_ld, y_ld;
    int64_t rows;
    int width;
    Shape shape;
    const void *pre, *post, *gate;  // null: ones
    int pre_code, post_code, gate_code;
    int64_t gate_rows;  // consecutive rows that share a gate row
    int post_norm;
    float scale, eps;
    void *x_new, *h;
    float* stats;  // [rows, 2]: r1, r2; null: not kept
    uint32_t* status;
};

template <int TX, int TY, bool VEC, bool WIDE, int SUBS>
__global__ void __launch_bounds__(MAX_WARPS * 32, FWD_RING<TX, TY, VEC> ? 1 : 2) norm_kernel(const NormArgs a) {
    constexpr int R = FWD_ROWS<TX, TY, VEC>, S = STAGES<TX, TY>, ROW = BYTES<TX> + BYTES<TY>;
    constexpr bool ringed = FWD_RING<TX, TY, VEC>;
    constexpr int MODE = mode_of(TX, TY, VEC);
    extern __shared__ float4 ring[];
    __shared__ float4 slots[SLOTS];
    __shared__ uint64_t filled[WIDE ? 2 : 1];
    using bx = typename Elt<TX>::bits;
    using by = typename Elt<TY>::bits;
    const int threads = blockDim.x, lane = threadIdx.x & 31, warps = a.shape.warps;
    const int group = (threadIdx.x >> 5) / warps, warp = (threadIdx.x >> 5) % warps;
    const int parts = WIDE ? a.shape.parts : 1, part = WIDE ? blockIdx.x % parts : 0;
    const int sub = SUBS > 1 ? lane / (32 / SUBS) : 0;  // which of the SUBS rows that the warp has side by side
    const Place<MODE> pl(warp, lane % (32 / SUBS), part * a.shape.cols, min(a.width, (part + 1) * a.shape.cols));
    for (int i = threadIdx.x; i < SLOTS; i += threads) slots[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if constexpr (WIDE) {
        if (threadIdx.x == 0) {
            mbar_init(&filled[0], 1);
            mbar_init(&filled[1], 1);
            fence_mbar_init();
        }
        cg::this_cluster().sync();
    } else {
        __syncthreads();
    }
    const int fold = fold_of(warps * parts);
    RowSums<R, WIDE, SUBS> sum(slots + group * 2 * fold, fold, warps, warp, lane, group + 1, parts, part, filled, a.status);
    const float inv_width = 1.0f / a.width;
    const int64_t begin = ((int64_t)(blockIdx.x / parts) * a.shape.groups + group) * a.shape.per;
    const int count = (int)max((int64_t)0, min(a.rows - begin, a.shape.per));
    const int rows = (count + SUBS - 1) / SUBS;  // of this lane, the last one perhaps behind the end
    auto row_of = [&](int r) { return (int64_t)r * SUBS + sub; };
    auto there = [&](int r) { return SUBS == 1 || r * SUBS + sub < count; };
    const bx* const px = reinterpret_cast<const bx*>(a.x) + begin * a.x_ld;
    const by* const py = reinterpret_cast<const by*>(a.y) + (a.y ? begin * a.y_ld : 0);
    bx* const po = reinterpret_cast<bx*>(a.x_new) + (a.x_new ? begin * a.width : 0);
    by* const ph = reinterpret_cast<by*>(a.h) + begin * a.width;
    const uint32_t base = (uint32_t)__cvta_generic_to_shared(ring);
    const uint32_t stage_bytes = ROW * R * threads, ring_end = base + S * stage_bytes;
    uint32_t to = base, from = base;
    int next = 0;  // row to copy
    auto ahead = [&]() {
#pragma unroll
        for (int k = 0; k < R; ++k)
            if (next + k < rows && there(next + k)) {
                const int64_t r = row_of(next + k);
                copy8<TX, MODE>(to + ROW * k * threads, threads, px + r * a.x_ld + pl.from, pl);
                if (a.y) copy8<TY, MODE>(to + (ROW * k + BYTES<TX>) * threads, threads, py + r * a.y_ld + pl.from, pl);
            }
        copy_commit();
        next += R;
        to = to + stage_bytes == ring_end ? base : to + stage_bytes;
    };
    if constexpr (ringed) {
        for (int i = 0; i < S * R; ++i) {
            clear8<TX, MODE>(base + ROW * i * threads, threads);
            clear8<TY, MODE>(base + (ROW * i + BYTES<TX>) * threads, threads);
        }
        for (int i = 1; i < S; ++i) ahead();
    }
    Pair pre[4], gain[4];  // gain: gate x post weight
    load_weight<MODE>(a.pre, a.pre_code, 0, pl, pre);
    load_scale<MODE>(nullptr, 0, 0, a.post, a.post_code, pl, gain);
    int gate_end = a.gate ? 0 : rows;  // the first row with another gate row than gain's
    for (int r0 = 0; r0 < rows; r0 += R) {
        if constexpr (ringed) {
            ahead();
            copy_wait<S - 1>();
        }
        int k0 = 0, k1;  // rows [k0, k1) of these share a gate row
        do {
            k1 = min(R, rows - r0);
            if (r0 + k0 >= gate_end) {
                const int64_t at = (begin + r0 + k0) / a.gate_rows;
                gate_end = (int)min((int64_t)rows, (at + 1) * a.gate_rows - begin);
                load_scale<MODE>(a.gate, a.gate_code, at * a.width, a.post, a.post_code, pl, gain);
            }
            k1 = min(k1, gate_end - r0);
            Pair x[R][4], y[R][4];
            float r1[R], t[R];
#pragma unroll
            for (int k = 0; k < R; ++k) {
                r1[k] = 1.f;
                Pair ss = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) y[k][i] = 0;
                if (a.y && k >= k0 && k < k1 && there(r0 + k)) {
                    if constexpr (ringed) take8<TY, MODE>(from + (ROW * k + BYTES<TX>) * threads, threads, y[k]);
                    else load8<TY, MODE>(py + row_of(r0 + k) * a.y_ld, pl, y[k]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) ss = fma2(y[k][i], y[k][i], ss);
                t[k] = sum_of(ss);
            }
            if (a.post_norm) {
                sum(t);
#pragma unroll
                for (int k = 0; k < R; ++k) r1[k] = rsqrtf(fmaf(t[k], inv_width, a.eps));
            }
#pragma unroll
            for (int k = 0; k < R; ++k) {
#pragma unroll
                for (int i = 0; i < 4; ++i) x[k][i] = 0;
                if (k >= k0 && k < k1 && there(r0 + k)) {
                    if constexpr (ringed) take8<TX, MODE>(from + ROW * k * threads, threads, x[k]);
                    else load8<TX, MODE>(px + row_of(r0 + k) * a.x_ld, pl, x[k]);
                    if (a.y) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            x[k][i] = fma2(gain[i], mul2(y[k][i], both(r1[k])), mul2(both(a.scale), x[k][i]));
                    }
                }
                Pair ss = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) ss = fma2(x[k][i], x[k][i], ss);
                t[k] = sum_of(ss);
            }
            sum(t);
#pragma unroll
            for (int k = 0; k < R; ++k) {
                if (k < k0 || k >= k1 || !there(r0 + k)) continue;
                if (a.y) store8<TX, MODE>(po + row_of(r0 + k) * a.width, pl, x[k]);
                t[k] = rsqrtf(fmaf(t[k], inv_width, a.eps));
#pragma unroll
                for (int i = 0; i < 4; ++i) x[k][i] = mul2(mul2(x[k][i], both(t[k])), pre[i]);
                store8<TY, MODE>(ph + row_of(r0 + k) * a.width, pl, x[k]);
                if (a.stats && part == 0 && warp == 0 && lane % (32 / SUBS) == 0)
                    reinterpret_cast<float2*>(a.stats)[begin + row_of(r0 + k)] = make_float2(r1[k], t[k]);
            }
            k0 = k1;
        } while (k0 < min(R, rows - r0));
        from = from + stage_bytes == ring_end ? base : from + stage_bytes;
    }
    if constexpr (WIDE) cg::this_cluster().sync();  // no block leaves while a fellow may write its slots
}

struct NormBwdArgs {
    const void *x, *y;
    int64_t x_ld, y_ld;
    int64_t rows;
    int width;
    Shape shape;
    const void *pre, *post, *gate;
    int pre_code, post_code, gate_code;
    int64_t gate_rows;
    int post_norm;
    float scale;
    const float* stats;
    const void *dx_new, *dh;  // null: zero
    void *dx, *dy;            // null: not wanted
    float* part;              // [blocks / parts][3][width]: dw_pre, dw_post, dgate (of one shared gate row)
    float* gate_part;         // [units + gate rows][width], where gates are not shared by all rows and a sum is wanted; else null
    int want;                 // bits 0..2: dw_pre, dw_post, dgate
    uint32_t* status;
};

enum { WANT_PRE = 1, WANT_POST = 2, WANT_GATE = 4 };

template <int TX, int TY, bool VEC, bool WIDE, int SUBS>
__global__ void __launch_bounds__(MAX_WARPS * 32, 1) norm_bwd_kernel(const NormBwdArgs a) {
    constexpr int S = BWD_STAGES<TX, TY>, ROW = 2 * (BYTES<TX> + BYTES<TY>);
    constexpr bool ringed = BWD_RING<TX, TY, VEC>;
    constexpr int MODE = mode_of(TX, TY, VEC);
    extern __shared__ float4 ring[];  // and, at the end, [groups][warps * 32][2]: the join of the block's groups
    __shared__ float4 slots[SLOTS];
    __shared__ uint64_t filled[WIDE ? 2 : 1];
    using bx = typename Elt<TX>::bits;
    using by = typename Elt<TY>::bits;
    const int threads = blockDim.x, lane = threadIdx.x & 31, warps = a.shape.warps;
    const int group = (threadIdx.x >> 5) / warps, warp = (threadIdx.x >> 5) % warps;
    const int parts = WIDE ? a.shape.parts : 1, part = WIDE ? blockIdx.x % parts : 0;
    const int sub = SUBS > 1 ? lane / (32 / SUBS) : 0;  // which of the SUBS rows that the warp has side by side
    const Place<MODE> pl(warp, lane % (32 / SUBS), part * a.shape.cols, min(a.width, (part + 1) * a.shape.cols));
    for (int i = threadIdx.x; i < SLOTS; i += threads) slots[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if constexpr (WIDE) {
        if (threadIdx.x == 0) {
            mbar_init(&filled[0], 1);
            mbar_init(&filled[1], 1);
            fence_mbar_init();
        }
        cg::this_cluster().sync();
    } else {
        __syncthreads();
    }
    const int fold = fold_of(warps * parts);
    RowSums<3, WIDE, SUBS> sum(slots + group * 2 * fold, fold, warps, warp, lane, group + 1, parts, part, filled, a.status);
    const float inv_width = 1.0f / a.width;
    const int64_t block = blockIdx.x / parts;
    const int64_t unit = block * a.shape.groups + group, begin = unit * a.shape.per;
    const int count = (int)max((int64_t)0, min(a.rows - begin, a.shape.per));
    const int rows = (count + SUBS - 1) / SUBS;  // of this lane, the last one perhaps behind the end
    auto there = [&](int r) { return SUBS == 1 || r * SUBS + sub < count; };
    const int64_t flat = (begin + sub) * a.width;  // of the contiguous arrays
    const bool has_x = a.dx_new != nullptr, has_y = a.y != nullptr, has_h = a.dh != nullptr;
    const bx* px = reinterpret_cast<const bx*>(a.x) + (begin + sub) * a.x_ld;
    const by* py = has_y ? reinterpret_cast<const by*>(a.y) + (begin + sub) * a.y_ld : nullptr;
    const bx* pe = has_x ? reinterpret_cast<const bx*>(a.dx_new) + flat : nullptr;
    const by* pt = has_h ? reinterpret_cast<const by*>(a.dh) + flat : nullptr;
    bx* po = a.dx ? reinterpret_cast<bx*>(a.dx) + flat : nullptr;
    by* pq = a.dy ? reinterpret_cast<by*>(a.dy) + flat : nullptr;
    const float2* stats = reinterpret_cast<const float2*>(a.stats) + begin + sub;
    const uint32_t base = (uint32_t)__cvta_generic_to_shared(ring);
    const uint32_t stage_bytes = ROW * threads, ring_end = base + S * stage_bytes;
    const uint32_t at_e = BYTES<TX> * threads, at_y = 2 * at_e, at_t = at_y + BYTES<TY> * threads;
    uint32_t to = base, from = base;
    int left = count - sub;  // to copy, at most
    const bx *cx = px + pl.from, *ce = pe + pl.from;  // of the next row to copy
    const by *cy = py + pl.from, *ct = pt + pl.from;
    auto ahead = [&]() {
        if (left > 0) {
            copy8<TX, MODE>(to, threads, cx, pl);
            if (has_x) copy8<TX, MODE>(to + at_e, threads, ce, pl);
            if (has_y) copy8<TY, MODE>(to + at_y, threads, cy, pl);
            if (has_h) copy8<TY, MODE>(to + at_t, threads, ct, pl);
        }
        copy_commit();
        left -= SUBS;
        cx += SUBS * a.x_ld;
        cy += SUBS * a.y_ld;
        ce += SUBS * a.width;
        ct += SUBS * a.width;
        to = to + stage_bytes == ring_end ? base : to + stage_bytes;
    };
    if constexpr (ringed) {
        for (int i = 0; i < S; ++i) {
            const uint32_t q = base + i * stage_bytes;
            clear8<TX, MODE>(q, threads);
            clear8<TX, MODE>(q + at_e, threads);
            clear8<TY, MODE>(q + at_y, threads);
            clear8<TY, MODE>(q + at_t, threads);
        }
        for (int i = 1; i < S; ++i) ahead();
    }
    Pair pre[4], gain[4], dpre[4], z[4], dpost[4];  // gain: gate x post weight; z: sum of e yh under one gate row
    load_weight<MODE>(a.pre, a.pre_code, 0, pl, pre);
    load_scale<MODE>(nullptr, 0, 0, a.post, a.post_code, pl, gain);
#pragma unroll
    for (int i = 0; i < 4; ++i) dpre[i] = z[i] = dpost[i] = 0;
    int gate_end = a.gate ? 0 : rows;  // the first row with another gate row than gain's, the gate_at-th
    int64_t gate_at = 0;
    float2 next = rows && there(0) ? stats[0] : make_float2(0.f, 0.f);
    for (int r = 0; r < rows; ++r) {
        const float r1 = next.x, r2 = next.y;
        if (r + 1 < rows && there(r + 1)) next = stats[(r + 1) * SUBS];
        if constexpr (ringed) ahead();
        if (r >= gate_end) {
            gate_at = (begin + r) / a.gate_rows;
            gate_end = (int)min((int64_t)rows, (gate_at + 1) * a.gate_rows - begin);
            load_scale<MODE>(a.gate, a.gate_code, gate_at * a.width, a.post, a.post_code, pl, gain);
        }
        Pair x[4], e[4], y[4], t[4];
        if constexpr (ringed) {
            copy_wait<S - 1>();
            take8<TX, MODE>(from, threads, x);
            take8<TX, MODE>(from + at_e, threads, e);
            take8<TY, MODE>(from + at_y, threads, y);
            take8<TY, MODE>(from + at_t, threads, t);
            from = from + stage_bytes == ring_end ? base : from + stage_bytes;
            if (!there(r))
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = e[i] = y[i] = t[i] = 0;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] = y[i] = t[i] = 0;
            load8<TX, MODE>(px, pl, x);
            if (has_x) load8<TX, MODE>(pe, pl, e);
            if (has_y) load8<TY, MODE>(py, pl, y);
            if (has_h) load8<TY, MODE>(pt, pl, t);
            px += a.x_ld;
            py += a.y_ld;
            pe += a.width;
            pt += a.width;
        }
        Pair s0 = 0, s1 = 0, s2 = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            y[i] = mul2(y[i], both(r1));  // yh
            const Pair q = mul2(gain[i], y[i]);
            x[i] = mul2(fma2(both(a.scale), x[i], q), both(r2));  // xh
            dpre[i] = fma2(t[i], x[i], dpre[i]);
            t[i] = mul2(t[i], pre[i]);
            e[i] = fma2(t[i], both(r2), e[i]);  // dx' + r2 t
            s0 = fma2(t[i], x[i], s0);
            s1 = fma2(q, e[i], s1);
            s2 = fma2(q, x[i], s2);
        }
        float v[3] = {sum_of(s0), sum_of(s1), sum_of(s2)};
        sum(v);
        const float c2 = r2 * (v[0] * inv_width);
        const float c1 = a.post_norm ? fmaf(-c2, v[2], v[1]) * inv_width : 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            e[i] = fma2(x[i], both(-c2), e[i]);
            x[i] = mul2(e[i], both(a.scale));
            z[i] = fma2(e[i], y[i], z[i]);
            e[i] = mul2(fma2(y[i], both(-c1), mul2(gain[i], e[i])), both(r1));
        }
        if (a.dx && there(r)) store8<TX, MODE>(po, pl, x);
        if (a.dy && there(r)) store8<TY, MODE>(pq, pl, e);
        po += SUBS * a.width;
        pq += SUBS * a.width;
        // the last of the unit's rows with this gate row: its sum goes out
        if (a.gate_part && r + 1 == gate_end) {
            Pair w[4];
            load_weight<MODE>(a.gate, a.gate_code, gate_at * a.width, pl, w);
#pragma unroll
            for (int i = 0; i < 4; ++i) dpost[i] = fma2(w[i], z[i], dpost[i]);
            load_weight<MODE>(a.post, a.post_code, 0, pl, w);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = mul2(w[i], z[i]);
            store8<SFFN_F32, MODE>(a.gate_part + (unit + gate_at) * a.width, pl, w);
#pragma unroll
            for (int i = 0; i < 4; ++i) z[i] = 0;
        }
    }
    if (!a.gate_part) {  // one gate row, or none, for all rows
        Pair w[4];
        load_weight<MODE>(a.gate, a.gate_code, 0, pl, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) dpost[i] = mul2(w[i], z[i]);
        load_weight<MODE>(a.post, a.post_code, 0, pl, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) z[i] = mul2(w[i], z[i]);  // dgate
    }
    // the sums of the rows side by side
#pragma unroll
    for (int o = 32 / SUBS; o < 32; o <<= 1)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            dpre[i] = add2(dpre[i], __shfl_xor_sync(FULL, dpre[i], o));
            dpost[i] = add2(dpost[i], __shfl_xor_sync(FULL, dpost[i], o));
            z[i] = add2(z[i], __shfl_xor_sync(FULL, z[i], o));
        }
    if constexpr (WIDE) cg::this_cluster().sync();  // no block leaves while a fellow may write its slots
    // The block's groups join their sums, in order, through the ring (whose copies
    // are done: the last waits left only empty groups); one row of each is written.
    // All threads add, a column's groups in order (one group after the other, with a
    // barrier each: 3000x128 13.2 us instead of 9.7, 32768x768 60.3 instead of 59.2).
    __syncthreads();
    const int groups = a.shape.groups, spread = warps * 32 * 2;  // float4 of a group
    auto put = [&](int which, Pair* d) {
        if (!((a.want >> which) & 1) || (which == 2 && a.gate_part)) return;
        float4* mine = ring + group * spread + (warp * 32 + lane) * 2;
        if (groups > 1) {
            float2 f[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = unpair(d[i]);
            mine[0] = make_float4(f[0].x, f[0].y, f[1].x, f[1].y);
            mine[1] = make_float4(f[2].x, f[2].y, f[3].x, f[3].y);
            __syncthreads();
            for (int e = threadIdx.x; e < spread; e += threads) {
                float4 f = ring[e];
                for (int g = 1; g < groups; ++g) {
                    const float4 p = ring[g * spread + e];
                    f.x += p.x; f.y += p.y; f.z += p.z; f.w += p.w;
                }
                ring[e] = f;
            }
            __syncthreads();
            if (group) return;
            const float4 p = mine[0], q = mine[1];
            d[0] = pair(p.x, p.y);
            d[1] = pair(p.z, p.w);
            d[2] = pair(q.x, q.y);
            d[3] = pair(q.z, q.w);
        }
        if (!sub) store8<SFFN_F32, MODE>(a.part + (block * 3 + which) * a.width, pl, d);
    };
    put(0, dpre);
    put(1, dpost);
    put(2, z);
}

// Joins the partial sums: blockIdx.y 0..2 the weight gradients (blocks rows of
// `part`), from 3 on a gate row each (the units that hold rows of it).  In 64 bits,
// rounded once: these are the largest sums of all, of the fewest terms.
struct JoinArgs {
    const float *part, *gate_part;
    int64_t blocks, units, per, gate_rows, rows;
    int width, want;
    void *dpre, *dpost, *dgate;
    int pre_code, post_code, gate_code;
};

template <int JOIN_ROWS>  // threads of a column
__global__ void __launch_bounds__(32 * JOIN_ROWS) norm_join_kernel(const JoinArgs a) {
    __shared__ double s[JOIN_ROWS][32];
    const int x = threadIdx.x, y = threadIdx.y;
    const int col = blockIdx.x * 32 + x;
    const int64_t gates = a.gate_part && a.dgate ? (a.rows + a.gate_rows - 1) / a.gate_rows : 0;
    for (int64_t which = blockIdx.y; which < 3 + gates; which += gridDim.y) {
        if (which < 3 && (!((a.want >> which) & 1) || (which == 2 && a.gate_part))) continue;
        // rows first .. last, `step` floats apart, of the sums
        const float* from = a.part + which * a.width;
        int64_t first = 0, last = a.blocks - 1, step = 3 * (int64_t)a.width;
        if (which >= 3) {  // the units that hold rows of gate row g
            const int64_t g = which - 3;
            from = a.gate_part + g * a.width;
            first = g * a.gate_rows / a.per;
            last = (min(a.rows, (g + 1) * a.gate_rows) - 1) / a.per;
            step = a.width;
        }
        double v = 0.0;
        if (col < a.width)
#pragma unroll 4
            for (int64_t u = first + y; u <= last; u += JOIN_ROWS) v += from[u * step + col];
        __syncthreads();
        s[y][x] = v;
        __syncthreads();
        if (y == 0 && col < a.width) {
            double all = 0.0;
#pragma unroll
            for (int i = 0; i < JOIN_ROWS; ++i) all += s[i][x];
            const float total = (float)all;
            if (which == 0) store_code(a.dpre, col, a.pre_code, total);
            else if (which == 1) store_code(a.dpost, col, a.post_code, total);
            else store_code(a.dgate, (which == 2 ? 0 : which - 3) * a.width + col, a.gate_code, total);
        }
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
constexpr int64_t MAX_WIDTH = (int64_t)MAX_PARTS * MAX_WARPS * 32 * CH;

// A block holds as many groups as make about 512 threads, but no more than there
// are rows (`at_a_time` of them to a group) for all SMs; one such block runs on
// an SM (128 registers a thread).  Of clusters of 4 blocks the SMs of one GPC
// hold 33 together, not 37: with 37 the last ones ran alone, in twice the time
// (bf16 4096x16384: 234 us forward, 397 backward; with 32 137 and 232).
Shape shape_of(int64_t rows, int64_t width, int at_a_time, int blocks_per_sm) {
    Shape s;
    const int64_t block_cols = MAX_WARPS * 32 * CH;
    s.parts = width <= block_cols ? 1 : width <= 2 * block_cols ? 2 : 4;
    s.cols = (int)((width + s.parts * CH - 1) / (s.parts * CH)) * CH;
    s.warps = (s.cols + 32 * CH - 1) / (32 * CH);
    s.groups = s.parts > 1 ? 1 : MAX_WARPS / s.warps;
    const int64_t share = rows / (SMS * at_a_time);
    if (share < s.groups) s.groups = (int)std::max<int64_t>(share, 1);
    const int64_t fit = s.parts == 4 ? 32 : SMS / s.parts;
    const int64_t most = fit * blocks_per_sm * (MAX_WARPS / (s.warps * s.groups));
    const int64_t want = (rows + s.groups - 1) / s.groups;
    const int64_t sets = want < most ? want : most;
    s.per = (rows + sets * s.groups - 1) / (sets * s.groups);
    s.blocks = sets * s.parts;
    return s;
}

// `smem_a_thread` bytes of dynamic shared memory.  The limit that a kernel carries
// is its device's and every host thread's, so it is always set to what the largest
// block takes: a smaller value, of a call with fewer threads, could come between
// another thread's set and launch.
template <class Args>
cudaError_t launch(void (*kernel)(Args), const Shape& s, int smem_a_thread, cudaStream_t st, const Args& a) {
    const int smem = smem_a_thread * s.threads(), most = smem_a_thread * MAX_WARPS * 32;
    if (smem > 32 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)s.blocks);
    cfg.blockDim = dim3((unsigned)s.threads());
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)s.parts;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = s.parts > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

struct Params {
    const void *pre, *post, *gate;
    int pre_code, post_code, gate_code;
};

int check_norm(int x_dtype, int y_dtype, int64_t rows, int64_t width, int64_t x_ld, bool has_y, int64_t y_ld,
               const Params& p, int64_t gate_rows) {
    if (!dtype_ok(x_dtype) || !dtype_ok(y_dtype)) return SFFN_ERR_DTYPE;
    if (x_dtype != y_dtype && x_dtype != SFFN_F32) return SFFN_ERR_DTYPE;
    if ((p.pre && !dtype_ok(p.pre_code)) || (p.post && !dtype_ok(p.post_code)) || (p.gate && !dtype_ok(p.gate_code)))
        return SFFN_ERR_DTYPE;
    if (rows < 0 || width < 1 || x_ld < 0 || (has_y && y_ld < 0) || (p.gate && gate_rows < 1)) return SFFN_ERR_ARG;
    if (!has_y && (p.post || p.gate)) return SFFN_ERR_ARG;
    if (width > MAX_WIDTH) return SFFN_ERR_TOO_LARGE;
    return SFFN_OK;
}

// Whether a pointer lies on its element's boundary.
bool lies(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % esize_of(dtype) == 0; }
bool lies8(const void* p) { return reinterpret_cast<uintptr_t>(p) % 8 == 0; }
bool row_aligned(const void* p, int64_t ld, int dtype) { return !p || (aligned16(p) && ld * esize_of(dtype) % 16 == 0); }

// Rows that a warp has side by side.  A row of at most 128 columns (float32, in
// either array: 64) leaves half of a warp's lanes idle, of 64 (16-bit types) three
// quarters, so two or four share the warp, where one gate row serves them all
// (forward, backward: bf16 100000x64 31 -> 12 and 46 -> 18 us, 200000x128 60 -> 39 and
// 84 -> 60; float32 100000x64 48 -> 27 and 50 -> 33).
int rows_a_warp(int64_t width, int x_dtype, bool vec, bool one_gate) {
    if (!vec || !one_gate) return 1;
    if (x_dtype == SFFN_F32) return width <= 64 ? 2 : 1;
    return width <= 64 ? 4 : width <= 128 ? 2 : 1;
}

template <class F>
int by_types(int x_dtype, int y_dtype, F&& f) {
    using std::integral_constant;
    if (x_dtype == SFFN_F32) {
        if (y_dtype == SFFN_F32) return f(integral_constant<int, SFFN_F32>(), integral_constant<int, SFFN_F32>());
        if (y_dtype == SFFN_BF16) return f(integral_constant<int, SFFN_F32>(), integral_constant<int, SFFN_BF16>());
        return f(integral_constant<int, SFFN_F32>(), integral_constant<int, SFFN_F16>());
    }
    if (x_dtype == SFFN_BF16) return f(integral_constant<int, SFFN_BF16>(), integral_constant<int, SFFN_BF16>());
    return f(integral_constant<int, SFFN_F16>(), integral_constant<int, SFFN_F16>());
}
}  // namespace
}  // namespace sffn

using namespace sffn;

extern "C" int sffn_residual_norm(const void* x, int x_dtype, int64_t x_ld, const void* y, int y_dtype, int64_t y_ld,
                                  int64_t rows, int64_t width, const void* pre, int pre_dtype, const void* post,
                                  int post_dtype, const void* gate, int gate_dtype, int64_t gate_rows,
                                  int post_norm, float scale, float eps, void* x_new, void* h, float* stats,
                                  uint32_t* status_dev, void* stream) {
    const Params p{pre, post, gate, pre_dtype, post_dtype, gate_dtype};
    if (int rc = check_norm(x_dtype, y_dtype, rows, width, x_ld, y != nullptr, y_ld, p, gate_rows)) return rc;
    if (!(eps > 0.f) || (post && !post_norm)) return SFFN_ERR_ARG;
    if (rows == 0) return SFFN_OK;
    if (!x || !h || (y && !x_new) || !status_dev) return SFFN_ERR_ARG;
    if (!lies(x, x_dtype) || !lies(y, y_dtype) || !lies(x_new, x_dtype) || !lies(h, y_dtype) || !lies(pre, pre_dtype) ||
        !lies(post, post_dtype) || !lies(gate, gate_dtype) || !lies8(stats))
        return SFFN_ERR_ALIGN;
    SFFN_BIND(scope, x);
    const bool vec = width % CH == 0 && row_aligned(x, x_ld, x_dtype) && row_aligned(y, y_ld, y_dtype) &&
                     row_aligned(x_new, width, x_dtype) && row_aligned(h, width, y_dtype) &&
                     row_aligned(pre, width, pre_dtype) && row_aligned(post, width, post_dtype) &&
                     row_aligned(gate, width, gate_dtype);
    const bool ringed = vec && (x_dtype != SFFN_F32 || y_dtype != SFFN_F32);
    const int subs = rows_a_warp(width, x_dtype, vec, !gate || gate_rows >= rows);
    const Shape s = ringed ? shape_of(rows, width, 4 * subs, 1) : shape_of(rows, width, 1, 2);
    const NormArgs a{x, y, x_ld, y_ld, rows, (int)width, s, pre, post, gate, pre_dtype, post_dtype, gate_dtype,
                     gate_rows, post_norm, scale, eps, x_new, h, stats, status_dev};
    return by_types(x_dtype, y_dtype, [&](auto tx, auto ty) -> int {
        constexpr int TX = decltype(tx)::value, TY = decltype(ty)::value;
        constexpr int FEW = TX == SFFN_F32 ? 2 : 4;
        SFFN_CUDA_TRY(launch(s.parts > 1 ? (vec ? norm_kernel<TX, TY, true, true, 1> : norm_kernel<TX, TY, false, true, 1>)
                             : subs == 4 ? norm_kernel<TX, TY, true, false, FEW>
                             : subs == 2 ? norm_kernel<TX, TY, true, false, 2>
                                         : (vec ? norm_kernel<TX, TY, true, false, 1> : norm_kernel<TX, TY, false, false, 1>), s,
                             ringed ? STAGES<TX, TY> * FWD_ROWS<TX, TY, true> * (BYTES<TX> + BYTES<TY>) : 0,
                             static_cast<cudaStream_t>(stream), a));
        return SFFN_OK;
    });
}

extern "C" size_t sffn_residual_norm_bwd_workspace_bytes(int64_t rows, int64_t width, int64_t gate_rows) {
    if (rows < 1 || width < 1 || width > MAX_WIDTH) return 0;
    const Shape s = shape_of(rows, width, 1, 1);
    int64_t n = s.blocks / s.parts * 3;
    if (gate_rows > 0 && gate_rows < rows) n += s.units() + (rows + gate_rows - 1) / gate_rows;
    return (size_t)(n * width) * sizeof(float);
}

extern "C" int sffn_residual_norm_bwd(const void* x, int x_dtype, int64_t x_ld, const void* y, int y_dtype,
                                      int64_t y_ld, int64_t rows, int64_t width, const void* pre, int pre_dtype,
                                      const void* post, int post_dtype, const void* gate, int gate_dtype,
                                      int64_t gate_rows, int post_norm, float scale, const float* stats,
                                      const void* dx_new, const void* dh, void* dx, void* dy, void* dpre,
                                      void* dpost, void* dgate, void* workspace, size_t workspace_bytes,
                                      uint32_t* status_dev, void* stream) {
    const Params p{pre, post, gate, pre_dtype, post_dtype, gate_dtype};
    if (int rc = check_norm(x_dtype, y_dtype, rows, width, x_ld, y != nullptr, y_ld, p, gate_rows)) return rc;
    if ((dpre && !pre) || (dpost && !post) || (dgate && !gate) || (dy && !y) || (post && !post_norm)) return SFFN_ERR_ARG;
    if (rows == 0) return SFFN_OK;
    if (!x || !stats || !status_dev) return SFFN_ERR_ARG;
    if (!lies(x, x_dtype) || !lies(y, y_dtype) || !lies(dx_new, x_dtype) || !lies(dh, y_dtype) || !lies(dx, x_dtype) ||
        !lies(dy, y_dtype) || !lies(pre, pre_dtype) || !lies(post, post_dtype) || !lies(gate, gate_dtype) ||
        !lies(dpre, pre_dtype) || !lies(dpost, post_dtype) || !lies(dgate, gate_dtype) || !lies8(stats))
        return SFFN_ERR_ALIGN;
    const bool shared_gate = !gate || gate_rows >= rows;
    const int want = (dpre ? WANT_PRE : 0) | (dpost ? WANT_POST : 0) | (dgate ? WANT_GATE : 0);
    const Shape s = shape_of(rows, width, 1, 1);
    if (want) {
        if (!workspace || !aligned16(workspace)) return SFFN_ERR_ALIGN;
        if (workspace_bytes < sffn_residual_norm_bwd_workspace_bytes(rows, width, dgate || dpost ? gate_rows : 0))
            return SFFN_ERR_WORKSPACE;
    }
    SFFN_BIND(scope, x);
    const bool vec = width % CH == 0 && row_aligned(x, x_ld, x_dtype) && row_aligned(y, y_ld, y_dtype) &&
                     row_aligned(dx_new, width, x_dtype) && row_aligned(dh, width, y_dtype) &&
                     row_aligned(dx, width, x_dtype) && row_aligned(dy, width, y_dtype) &&
                     row_aligned(pre, width, pre_dtype) && row_aligned(post, width, post_dtype) &&
                     row_aligned(gate, width, gate_dtype);
    const int subs = rows_a_warp(width, x_dtype, vec, shared_gate);
    float* part = static_cast<float*>(workspace);
    const int64_t sets = s.blocks / s.parts;
    float* gate_part = (dgate || dpost) && !shared_gate ? part + sets * 3 * width : nullptr;
    const NormBwdArgs a{x, y, x_ld, y_ld, rows, (int)width, s, pre, post, gate, pre_dtype, post_dtype, gate_dtype,
                        gate_rows, post_norm, y ? scale : 1.0f, stats, dx_new, dh, dx, dy, part, gate_part, want,
                        status_dev};
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int rc = by_types(x_dtype, y_dtype, [&](auto tx, auto ty) -> int {
        constexpr int TX = decltype(tx)::value, TY = decltype(ty)::value;
        constexpr int FEW = TX == SFFN_F32 ? 2 : 4;
        SFFN_CUDA_TRY(launch(s.parts > 1 ? (vec ? norm_bwd_kernel<TX, TY, true, true, 1> : norm_bwd_kernel<TX, TY, false, true, 1>)
                             : subs == 4 ? norm_bwd_kernel<TX, TY, true, false, FEW>
                             : subs == 2 ? norm_bwd_kernel<TX, TY, true, false, 2>
                                         : (vec ? norm_bwd_kernel<TX, TY, true, false, 1> : norm_bwd_kernel<TX, TY, false, false, 1>), s,
                             vec || BWD_RING<TX, TY, false> ? BWD_STAGES<TX, TY> * 2 * (BYTES<TX> + BYTES<TY>) : 32,
                             st, a));
        return SFFN_OK;
    });
    if (rc) return rc;
    if (want) {
        const JoinArgs j{part, gate_part, sets, s.units(), s.per, gate_rows, rows, (int)width, want,
                         dpre, dpost, dgate, pre_dtype, post_dtype, gate_dtype};
        const int64_t gates = gate_part ? (rows + gate_rows - 1) / gate_rows : 0;
        const int64_t ny = 3 + gates < 65535 ? 3 + gates : 65535;
        // Where the columns fill the SMs 8 threads add one up (the whole backward of
        // 8192x8192 with 8 gate rows: 237 us, with 32 threads 273); fewer columns take
        // 32, whose loads are in flight together (32768x768: 2 us less than with 8).
        const dim3 grid((unsigned)((width + 31) / 32), (unsigned)ny);
        if ((int64_t)grid.x * grid.y >= 4 * SMS) norm_join_kernel<8><<<grid, dim3(32, 8), 0, st>>>(j);
        else norm_join_kernel<32><<<grid, dim3(32, 32), 0, st>>>(j);
        SFFN_CHECK_LAUNCH();
    }
    return SFFN_OK;
}
