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
//   dw_pre = sum dh xh, dw_post = sum du yh, dgate = sum e u   (over the rows)
// x' is recomputed from x and y in the backward, unrounded, for the bytes that
// reading it back would take.  All arithmetic, the row statistics and the sums
// over rows are float32; each output is rounded once.
//
// Bound by memory: the forward moves four arrays of the stream's size, the
// backward six.  A row stays in the registers of one group of warps from its
// load to its stores.  The weight gradients are summed over a group's rows in
// registers (shared memory from two chunks a thread on, where they would
// spill), written once per block and joined by a second, small kernel in a
// fixed order, so equal inputs give equal bits.
#include <math.h>

#include "common.cuh"

namespace sffn {
namespace {

constexpr int CH = 8;          // elements of a thread's chunk
constexpr int MAX_WARPS = 16;  // warps that share a row
constexpr int SMS = 148;

__device__ __forceinline__ void store_code(void* p, int64_t i, int code, float v) {
    if (code == SFFN_F32) reinterpret_cast<float*>(p)[i] = v;
    else if (code == SFFN_BF16) reinterpret_cast<uint16_t*>(p)[i] = Elt<SFFN_BF16>::from_f(v);
    else reinterpret_cast<uint16_t*>(p)[i] = Elt<SFFN_F16>::from_f(v);
}

// A thread's place in its group and the columns of its chunks: with VEC eight
// neighbours (16-byte accesses), else every 32nd column of a warp's 256, so
// that single-element accesses of a warp stay together.
template <bool VEC>
struct Place {
    int warps, wg, lane, width;
    __device__ __forceinline__ int col(int v, int j) const {
        return VEC ? ((v * warps + wg) * 32 + lane) * CH + j : (v * warps + wg) * 32 * CH + j * 32 + lane;
    }
};

template <int DT, bool VEC>
__device__ __forceinline__ void load8(const void* base, const Place<VEC>& pl, int v, float* x) {
    using bits = typename Elt<DT>::bits;
    const bits* p = reinterpret_cast<const bits*>(base);
    if constexpr (VEC) {
        const int c = pl.col(v, 0);
        if (c < pl.width) {
            if constexpr (DT == SFFN_F32) {
                const float4 a = *reinterpret_cast<const float4*>(p + c), b = *reinterpret_cast<const float4*>(p + c + 4);
                x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
                x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
            } else {
                const uint4 q = *reinterpret_cast<const uint4*>(p + c);
                const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[2 * i] = Elt<DT>::to_f((uint16_t)u[i]);
                    x[2 * i + 1] = Elt<DT>::to_f((uint16_t)(u[i] >> 16));
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < CH; ++j) x[j] = 0.f;
        }
    } else {
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            const int c = pl.col(v, j);
            x[j] = c < pl.width ? Elt<DT>::to_f(p[c]) : 0.f;
        }
    }
}

// The same of a weight or gate row, whose type is an argument.
template <bool VEC>
__device__ __forceinline__ void load_weight(const void* p, int code, int64_t offset, const Place<VEC>& pl, int v,
                                            float* x) {
    if (code == SFFN_F32) load8<SFFN_F32, VEC>(reinterpret_cast<const float*>(p) + offset, pl, v, x);
    else if (code == SFFN_BF16) load8<SFFN_BF16, VEC>(reinterpret_cast<const uint16_t*>(p) + offset, pl, v, x);
    else load8<SFFN_F16, VEC>(reinterpret_cast<const uint16_t*>(p) + offset, pl, v, x);
}

template <int DT, bool VEC>
__device__ __forceinline__ void store8(void* base, const Place<VEC>& pl, int v, const float* x) {
    using bits = typename Elt<DT>::bits;
    bits* p = reinterpret_cast<bits*>(base);
    if constexpr (VEC) {
        const int c = pl.col(v, 0);
        if (c < pl.width) {
            if constexpr (DT == SFFN_F32) {
                *reinterpret_cast<float4*>(p + c) = make_float4(x[0], x[1], x[2], x[3]);
                *reinterpret_cast<float4*>(p + c + 4) = make_float4(x[4], x[5], x[6], x[7]);
            } else {
                uint32_t u[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    u[i] = (uint32_t)Elt<DT>::from_f(x[2 * i]) | ((uint32_t)Elt<DT>::from_f(x[2 * i + 1]) << 16);
                *reinterpret_cast<uint4*>(p + c) = make_uint4(u[0], u[1], u[2], u[3]);
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            const int c = pl.col(v, j);
            if (c < pl.width) p[c] = Elt<DT>::from_f(x[j]);
        }
    }
}

// Sum over a group's warps.  Two slot sets alternate: a set is written again
// only after the other set's barrier, which every reader of it has passed.
struct GroupSum {
    float* slots;  // this group's [2][MAX_WARPS]
    int warps, wg, lane, bar;
    int turn;
    __device__ __forceinline__ float operator()(float v) {
#pragma unroll
        for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
        if (warps == 1) return v;
        float* s = slots + turn * MAX_WARPS;
        turn ^= 1;
        if (lane == 0) s[wg] = v;
        asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(warps * 32) : "memory");
        float r = 0.f;
        for (int i = 0; i < warps; ++i) r += s[i];
        return r;
    }
};

struct NormArgs {
    const void *x, *y;  // y null: no block output, h = norm of x alone
    int64_t x_ld, y_ld;
    int64_t rows;
    int width, warps, groups;
    const void *pre, *post, *gate;  // null: ones
    int pre_code, post_code, gate_code;
    int64_t gate_rows;  // consecutive rows that share a gate row
    int post_norm;
    float scale, eps;
    void *x_new, *h;
    float* stats;  // [rows, 2]: r1, r2; null: not kept
};

template <int TX, int TY, int V, bool VEC>
__global__ void __launch_bounds__(MAX_WARPS * 32) norm_kernel(const NormArgs a) {
    __shared__ float slots[8][2 * MAX_WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = warp / a.warps;
    const Place<VEC> pl{a.warps, warp % a.warps, lane, a.width};
    GroupSum sum{slots[group], a.warps, pl.wg, lane, group + 1, 0};
    const float inv_width = 1.0f / a.width;
    using bx = typename Elt<TX>::bits;
    using by = typename Elt<TY>::bits;
    for (int64_t r = (int64_t)blockIdx.x * a.groups + group; r < a.rows; r += (int64_t)gridDim.x * a.groups) {
        float x[V][CH];
#pragma unroll
        for (int v = 0; v < V; ++v) load8<TX, VEC>(reinterpret_cast<const bx*>(a.x) + r * a.x_ld, pl, v, x[v]);
        float r1 = 1.f;
        if (a.y) {
            float y[V][CH];
#pragma unroll
            for (int v = 0; v < V; ++v) load8<TY, VEC>(reinterpret_cast<const by*>(a.y) + r * a.y_ld, pl, v, y[v]);
            if (a.post_norm) {
                float ss = 0.f;
#pragma unroll
                for (int v = 0; v < V; ++v)
#pragma unroll
                    for (int j = 0; j < CH; ++j) ss = fmaf(y[v][j], y[v][j], ss);
                r1 = rsqrtf(sum(ss) * inv_width + a.eps);
            }
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float w[CH], g[CH];
#pragma unroll
                for (int j = 0; j < CH; ++j) w[j] = g[j] = 1.f;
                if (a.post) load_weight<VEC>(a.post, a.post_code, 0, pl, v, w);
                if (a.gate) load_weight<VEC>(a.gate, a.gate_code, r / a.gate_rows * a.width, pl, v, g);
#pragma unroll
                for (int j = 0; j < CH; ++j) x[v][j] = fmaf(g[j], y[v][j] * r1 * w[j], a.scale * x[v][j]);
                store8<TX, VEC>(reinterpret_cast<bx*>(a.x_new) + r * a.width, pl, v, x[v]);
            }
        }
        float ss = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int j = 0; j < CH; ++j) ss = fmaf(x[v][j], x[v][j], ss);
        const float r2 = rsqrtf(sum(ss) * inv_width + a.eps);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float w[CH];
#pragma unroll
            for (int j = 0; j < CH; ++j) w[j] = 1.f;
            if (a.pre) load_weight<VEC>(a.pre, a.pre_code, 0, pl, v, w);
#pragma unroll
            for (int j = 0; j < CH; ++j) w[j] *= x[v][j] * r2;
            store8<TY, VEC>(reinterpret_cast<by*>(a.h) + r * a.width, pl, v, w);
        }
        if (a.stats && pl.wg == 0 && lane == 0) {
            a.stats[2 * r] = r1;
            a.stats[2 * r + 1] = r2;
        }
    }
}

struct NormBwdArgs {
    const void *x, *y;
    int64_t x_ld, y_ld;
    int64_t rows;
    int width, warps, groups;
    const void *pre, *post, *gate;
    int pre_code, post_code, gate_code;
    int64_t gate_rows;
    int post_norm;
    float scale;
    const float* stats;
    const void *dx_new, *dh;  // null: zero
    void *dx, *dy;            // null: not wanted
    int64_t per;              // consecutive rows of one group
    float* part;              // [blocks][3][width]: dw_pre, dw_post, dgate (of one shared gate row)
    float* gate_part;         // [units + gate rows][width], where gates are not shared by all rows; else null
    int want;                 // bits 0..2: dw_pre, dw_post, dgate
};

enum { WANT_PRE = 1, WANT_POST = 2, WANT_GATE = 4 };

// Sums over rows of one thread's columns: registers with one chunk a thread,
// else shared memory laid out so that a warp's accesses are 16 bytes a lane.
template <int V>
struct Sums {
    static constexpr bool SHARED = V > 1;
    float r[SHARED ? 1 : 3][CH];
    float4* s;
    int threads;
    __device__ __forceinline__ float4* at(int which, int v, int half) const {
        return s + ((which * V + v) * 2 + half) * threads + threadIdx.x;
    }
    __device__ __forceinline__ void clear(int which) {
        if constexpr (SHARED) {
#pragma unroll
            for (int v = 0; v < V; ++v) *at(which, v, 0) = *at(which, v, 1) = make_float4(0.f, 0.f, 0.f, 0.f);
        } else {
#pragma unroll
            for (int j = 0; j < CH; ++j) r[which][j] = 0.f;
        }
    }
    __device__ __forceinline__ void add(int which, int v, const float* d) {
        if constexpr (SHARED) {
            float4 p = *at(which, v, 0), q = *at(which, v, 1);
            p.x += d[0]; p.y += d[1]; p.z += d[2]; p.w += d[3];
            q.x += d[4]; q.y += d[5]; q.z += d[6]; q.w += d[7];
            *at(which, v, 0) = p;
            *at(which, v, 1) = q;
        } else {
#pragma unroll
            for (int j = 0; j < CH; ++j) r[which][j] += d[j];
        }
    }
    __device__ __forceinline__ void get(int which, int v, float* d) const {
        if constexpr (SHARED) {
            const float4 p = *at(which, v, 0), q = *at(which, v, 1);
            d[0] = p.x; d[1] = p.y; d[2] = p.z; d[3] = p.w;
            d[4] = q.x; d[5] = q.y; d[6] = q.z; d[7] = q.w;
        } else {
#pragma unroll
            for (int j = 0; j < CH; ++j) d[j] = r[which][j];
        }
    }
};

template <int TX, int TY, int V, bool VEC>
__global__ void __launch_bounds__(MAX_WARPS * 32) norm_bwd_kernel(const NormBwdArgs a) {
    extern __shared__ float4 dyn[];  // V > 1: the sums; else the block's join
    __shared__ float slots[8][2 * MAX_WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = warp / a.warps;
    const Place<VEC> pl{a.warps, warp % a.warps, lane, a.width};
    GroupSum sum{slots[group], a.warps, pl.wg, lane, group + 1, 0};
    Sums<V> acc;
    acc.s = dyn;
    acc.threads = blockDim.x;
#pragma unroll
    for (int w = 0; w < 3; ++w) acc.clear(w);
    const float inv_width = 1.0f / a.width;
    using bx = typename Elt<TX>::bits;
    using by = typename Elt<TY>::bits;
    const int64_t unit = (int64_t)blockIdx.x * a.groups + group;
    const int64_t end = min(a.rows, (unit + 1) * a.per);
    for (int64_t r = unit * a.per; r < end; ++r) {
        float x[V][CH], y[V][CH], t[V][CH], e[V][CH];
        const float r1 = a.stats[2 * r], r2 = a.stats[2 * r + 1];
        const int64_t gate_at = a.gate ? r / a.gate_rows : 0;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            load8<TX, VEC>(reinterpret_cast<const bx*>(a.x) + r * a.x_ld, pl, v, x[v]);
            if (a.y) load8<TY, VEC>(reinterpret_cast<const by*>(a.y) + r * a.y_ld, pl, v, y[v]);
            if (a.dh) load8<TY, VEC>(reinterpret_cast<const by*>(a.dh) + r * a.width, pl, v, t[v]);
            if (a.dx_new) load8<TX, VEC>(reinterpret_cast<const bx*>(a.dx_new) + r * a.width, pl, v, e[v]);
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                if (!a.dh) t[v][j] = 0.f;
                if (!a.dx_new) e[v][j] = 0.f;
            }
        }
        float dot = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float w[CH], g[CH];
            if (a.y) {
#pragma unroll
                for (int j = 0; j < CH; ++j) w[j] = g[j] = 1.f;
                if (a.post) load_weight<VEC>(a.post, a.post_code, 0, pl, v, w);
                if (a.gate) load_weight<VEC>(a.gate, a.gate_code, gate_at * a.width, pl, v, g);
#pragma unroll
                for (int j = 0; j < CH; ++j) {
                    y[v][j] *= r1;
                    x[v][j] = fmaf(g[j], y[v][j] * w[j], a.scale * x[v][j]);
                }
            }
#pragma unroll
            for (int j = 0; j < CH; ++j) x[v][j] *= r2;  // xh
            if (a.want & WANT_PRE) {
#pragma unroll
                for (int j = 0; j < CH; ++j) w[j] = t[v][j] * x[v][j];
                acc.add(0, v, w);
            }
            if (a.pre) {
                load_weight<VEC>(a.pre, a.pre_code, 0, pl, v, w);
#pragma unroll
                for (int j = 0; j < CH; ++j) t[v][j] *= w[j];
            }
#pragma unroll
            for (int j = 0; j < CH; ++j) dot = fmaf(t[v][j], x[v][j], dot);
        }
        const float mean = sum(dot) * inv_width;
        float dot1 = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float w[CH], g[CH];
#pragma unroll
            for (int j = 0; j < CH; ++j) e[v][j] = fmaf(r2, t[v][j] - x[v][j] * mean, e[v][j]);
            if (a.dx) {
#pragma unroll
                for (int j = 0; j < CH; ++j) w[j] = a.y ? a.scale * e[v][j] : e[v][j];
                store8<TX, VEC>(reinterpret_cast<bx*>(a.dx) + r * a.width, pl, v, w);
            }
            if (!a.y) continue;
#pragma unroll
            for (int j = 0; j < CH; ++j) w[j] = g[j] = 1.f;
            if (a.post) load_weight<VEC>(a.post, a.post_code, 0, pl, v, w);
            if (a.gate) load_weight<VEC>(a.gate, a.gate_code, gate_at * a.width, pl, v, g);
            if (a.want & WANT_GATE) {
                float d[CH];
#pragma unroll
                for (int j = 0; j < CH; ++j) d[j] = e[v][j] * y[v][j] * w[j];
                acc.add(2, v, d);
            }
#pragma unroll
            for (int j = 0; j < CH; ++j) e[v][j] *= g[j];  // du
            if (a.want & WANT_POST) {
#pragma unroll
                for (int j = 0; j < CH; ++j) g[j] = e[v][j] * y[v][j];
                acc.add(1, v, g);
            }
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                e[v][j] *= w[j];  // the gradient of y r1
                dot1 = fmaf(e[v][j], y[v][j], dot1);
            }
        }
        if (a.y && a.dy) {
            const float mean1 = a.post_norm ? sum(dot1) * inv_width : 0.f;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float d[CH];
#pragma unroll
                for (int j = 0; j < CH; ++j) d[j] = r1 * (e[v][j] - y[v][j] * mean1);
                store8<TY, VEC>(reinterpret_cast<by*>(a.dy) + r * a.width, pl, v, d);
            }
        }
        // the last of the unit's rows with this gate row: its sum goes out
        if (a.gate_part && (r + 1 == end || (r + 1) / a.gate_rows != gate_at)) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float d[CH];
                acc.get(2, v, d);
                store8<SFFN_F32, VEC>(a.gate_part + (unit + gate_at) * a.width, pl, v, d);
            }
            acc.clear(2);
        }
    }
    // The block's groups join their sums in order; one row of each is written.
    if constexpr (V > 1) {  // one group
#pragma unroll
        for (int w = 0; w < 3; ++w) {
            if (!((a.want >> w) & 1) || (w == 2 && a.gate_part)) continue;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float d[CH];
                acc.get(w, v, d);
                store8<SFFN_F32, VEC>(a.part + ((int64_t)blockIdx.x * 3 + w) * a.width, pl, v, d);
            }
        }
    } else {
        float4* mine = dyn + (pl.wg * 32 + lane) * 2;  // the same place for the same columns of every group
#pragma unroll
        for (int w = 0; w < 3; ++w) {
            if (!((a.want >> w) & 1) || (w == 2 && a.gate_part)) continue;
            for (int g = 0; g < a.groups; ++g) {
                __syncthreads();
                if (group != g) continue;
                float d[CH];
                acc.get(w, 0, d);
                if (g) {
                    const float4 p = mine[0], q = mine[1];
                    d[0] += p.x; d[1] += p.y; d[2] += p.z; d[3] += p.w;
                    d[4] += q.x; d[5] += q.y; d[6] += q.z; d[7] += q.w;
                }
                if (g + 1 < a.groups) {
                    mine[0] = make_float4(d[0], d[1], d[2], d[3]);
                    mine[1] = make_float4(d[4], d[5], d[6], d[7]);
                } else {
                    store8<SFFN_F32, VEC>(a.part + ((int64_t)blockIdx.x * 3 + w) * a.width, pl, 0, d);
                }
            }
        }
    }
}

// Joins the partial sums: blockIdx.y 0..2 the weight gradients (blocks rows of
// `part`), from 3 on a gate row each (the units that hold rows of it).
struct JoinArgs {
    const float *part, *gate_part;
    int64_t blocks, units, per, gate_rows, rows;
    int width, want;
    void *dpre, *dpost, *dgate;
    int pre_code, post_code, gate_code;
};

__global__ void norm_join_kernel(const JoinArgs a) {
    __shared__ float s[32][33];
    const int x = threadIdx.x, y = threadIdx.y;
    const int col = blockIdx.x * 32 + x;
    for (int64_t which = blockIdx.y; which < 3 + (a.gate_part ? (a.rows + a.gate_rows - 1) / a.gate_rows : 0);
         which += gridDim.y) {
        if (which < 3 && (!((a.want >> which) & 1) || (which == 2 && a.gate_part))) continue;
        float v = 0.f;
        if (col < a.width) {
            if (which < 3) {
                for (int64_t b = y; b < a.blocks; b += 32) v += a.part[(b * 3 + which) * a.width + col];
            } else {
                const int64_t g = which - 3;
                const int64_t first = g * a.gate_rows / a.per, last = (min(a.rows, (g + 1) * a.gate_rows) - 1) / a.per;
                for (int64_t u = first + y; u <= last; u += 32) v += a.gate_part[(u + g) * a.width + col];
            }
        }
        __syncthreads();
        s[y][x] = v;
        __syncthreads();
        if (y == 0 && col < a.width) {
            float total = 0.f;
#pragma unroll
            for (int i = 0; i < 32; ++i) total += s[i][x];
            if (which == 0) store_code(a.dpre, col, a.pre_code, total);
            else if (which == 1) store_code(a.dpost, col, a.post_code, total);
            else store_code(a.dgate, (which == 2 ? 0 : which - 3) * a.width + col, a.gate_code, total);
        }
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
constexpr int64_t MAX_WIDTH = (int64_t)MAX_WARPS * 32 * CH * 4;  // four chunks a thread

struct Shape {
    int chunks, warps, groups;
    int64_t blocks, per;  // blocks of the launch; backward: rows of one group
    int threads() const { return warps * groups * 32; }
};

Shape shape_of(int64_t rows, int64_t width) {
    Shape s;
    const int64_t lanes = (width + CH - 1) / CH;
    s.chunks = lanes <= MAX_WARPS * 32 ? 1 : lanes <= MAX_WARPS * 32 * 2 ? 2 : 4;
    s.warps = (int)((lanes + 32 * s.chunks - 1) / (32 * s.chunks));
    s.groups = s.warps >= 8 ? 1 : 8 / s.warps;
    const int64_t most = (int64_t)SMS * (s.threads() > 256 ? 2 : 4);
    const int64_t want = (rows + s.groups - 1) / s.groups;
    s.blocks = want < most ? want : most;
    s.per = s.blocks ? (rows + s.blocks * s.groups - 1) / (s.blocks * s.groups) : 1;
    return s;
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

bool row_aligned(const void* p, int64_t ld, int dtype) { return !p || (aligned16(p) && ld * esize_of(dtype) % 16 == 0); }

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
template <class F>
int by_chunks(int chunks, bool vec, F&& f) {
    using std::integral_constant;
    if (vec) {
        if (chunks == 1) return f(integral_constant<int, 1>(), std::true_type());
        if (chunks == 2) return f(integral_constant<int, 2>(), std::true_type());
        return f(integral_constant<int, 4>(), std::true_type());
    }
    if (chunks == 1) return f(integral_constant<int, 1>(), std::false_type());
    if (chunks == 2) return f(integral_constant<int, 2>(), std::false_type());
    return f(integral_constant<int, 4>(), std::false_type());
}

}  // namespace
}  // namespace sffn

using namespace sffn;

extern "C" int sffn_residual_norm(const void* x, int x_dtype, int64_t x_ld, const void* y, int y_dtype, int64_t y_ld,
                                  int64_t rows, int64_t width, const void* pre, int pre_dtype, const void* post,
                                  int post_dtype, const void* gate, int gate_dtype, int64_t gate_rows,
                                  int post_norm, float scale, float eps, void* x_new, void* h, float* stats,
                                  void* stream) {
    const Params p{pre, post, gate, pre_dtype, post_dtype, gate_dtype};
    if (int rc = check_norm(x_dtype, y_dtype, rows, width, x_ld, y != nullptr, y_ld, p, gate_rows)) return rc;
    if (!(eps > 0.f) || (post && !post_norm)) return SFFN_ERR_ARG;
    if (rows == 0) return SFFN_OK;
    if (!x || !h || (y && !x_new)) return SFFN_ERR_ARG;
    SFFN_BIND(scope, x);
    const Shape s = shape_of(rows, width);
    const bool vec = width % CH == 0 && row_aligned(x, x_ld, x_dtype) && row_aligned(y, y_ld, y_dtype) &&
                     row_aligned(x_new, width, x_dtype) && row_aligned(h, width, y_dtype) &&
                     row_aligned(pre, width, pre_dtype) && row_aligned(post, width, post_dtype) &&
                     row_aligned(gate, width, gate_dtype);
    const NormArgs a{x, y, x_ld, y_ld, rows, (int)width, s.warps, s.groups, pre, post, gate, pre_dtype, post_dtype,
                     gate_dtype, gate_rows, post_norm, scale, eps, x_new, h, stats};
    by_types(x_dtype, y_dtype, [&](auto tx, auto ty) {
        return by_chunks(s.chunks, vec, [&](auto v, auto aligned) {
            norm_kernel<decltype(tx)::value, decltype(ty)::value, decltype(v)::value, decltype(aligned)::value>
                <<<(unsigned)s.blocks, s.threads(), 0, static_cast<cudaStream_t>(stream)>>>(a);
            return 0;
        });
    });
    SFFN_CHECK_LAUNCH();
    return SFFN_OK;
}

extern "C" size_t sffn_residual_norm_bwd_workspace_bytes(int64_t rows, int64_t width, int64_t gate_rows) {
    if (rows < 1 || width < 1 || width > MAX_WIDTH) return 0;
    const Shape s = shape_of(rows, width);
    int64_t n = s.blocks * 3;
    if (gate_rows > 0 && gate_rows < rows) n += s.blocks * s.groups + (rows + gate_rows - 1) / gate_rows;
    return (size_t)(n * width) * sizeof(float);
}

extern "C" int sffn_residual_norm_bwd(const void* x, int x_dtype, int64_t x_ld, const void* y, int y_dtype,
                                      int64_t y_ld, int64_t rows, int64_t width, const void* pre, int pre_dtype,
                                      const void* post, int post_dtype, const void* gate, int gate_dtype,
                                      int64_t gate_rows, int post_norm, float scale, const float* stats,
                                      const void* dx_new, const void* dh, void* dx, void* dy, void* dpre,
                                      void* dpost, void* dgate, void* workspace, size_t workspace_bytes,
                                      void* stream) {
    const Params p{pre, post, gate, pre_dtype, post_dtype, gate_dtype};
    if (int rc = check_norm(x_dtype, y_dtype, rows, width, x_ld, y != nullptr, y_ld, p, gate_rows)) return rc;
    if ((dpre && !pre) || (dpost && !post) || (dgate && !gate) || (dy && !y) || (post && !post_norm)) return SFFN_ERR_ARG;
    if (rows == 0) return SFFN_OK;
    if (!x || !stats) return SFFN_ERR_ARG;
    const bool shared_gate = !gate || gate_rows >= rows;
    const int want = (dpre ? WANT_PRE : 0) | (dpost ? WANT_POST : 0) | (dgate ? WANT_GATE : 0);
    const Shape s = shape_of(rows, width);
    if (want) {
        if (!workspace || !aligned16(workspace)) return SFFN_ERR_ALIGN;
        if (workspace_bytes < sffn_residual_norm_bwd_workspace_bytes(rows, width, dgate ? gate_rows : 0))
            return SFFN_ERR_WORKSPACE;
    }
    SFFN_BIND(scope, x);
    const bool vec = width % CH == 0 && row_aligned(x, x_ld, x_dtype) && row_aligned(y, y_ld, y_dtype) &&
                     row_aligned(dx_new, width, x_dtype) && row_aligned(dh, width, y_dtype) &&
                     row_aligned(dx, width, x_dtype) && row_aligned(dy, width, y_dtype) &&
                     row_aligned(pre, width, pre_dtype) && row_aligned(post, width, post_dtype) &&
                     row_aligned(gate, width, gate_dtype);
    float* part = static_cast<float*>(workspace);
    float* gate_part = dgate && !shared_gate ? part + s.blocks * 3 * width : nullptr;
    const NormBwdArgs a{x, y, x_ld, y_ld, rows, (int)width, s.warps, s.groups, pre, post, gate, pre_dtype, post_dtype,
                        gate_dtype, gate_rows, post_norm, scale, stats, dx_new, dh, dx, dy, s.per, part, gate_part,
                        want};
    const size_t smem = s.chunks > 1 ? (size_t)3 * s.chunks * 2 * s.threads() * 16 : (size_t)s.warps * 32 * 32;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int rc = by_types(x_dtype, y_dtype, [&](auto tx, auto ty) {
        return by_chunks(s.chunks, vec, [&](auto v, auto aligned) -> int {
            auto* k = norm_bwd_kernel<decltype(tx)::value, decltype(ty)::value, decltype(v)::value,
                                      decltype(aligned)::value>;
            if (smem > 32 * 1024)
                SFFN_CUDA_TRY(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
            k<<<(unsigned)s.blocks, s.threads(), smem, st>>>(a);
            return SFFN_OK;
        });
    });
    if (rc) return rc;
    SFFN_CHECK_LAUNCH();
    if (want) {
        const JoinArgs j{part, gate_part, s.blocks, s.blocks * s.groups, s.per, gate_rows, rows, (int)width, want,
                         dpre, dpost, dgate, pre_dtype, post_dtype, gate_dtype};
        const int64_t gates = gate_part ? (rows + gate_rows - 1) / gate_rows : 0;
        const int64_t ny = 3 + gates < 65535 ? 3 + gates : 65535;
        norm_join_kernel<<<dim3((unsigned)((width + 31) / 32), (unsigned)ny), dim3(32, 32), 0, st>>>(j);
        SFFN_CHECK_LAUNCH();
    }
    return SFFN_OK;
}
