// ckpt_linear and the gated feed-forward block as one call a direction: operands
// whose rows are not on 16 bytes copied (one launch for all of them), the
// products, the 8-bit checkpoints.  A training step of a small layer is bound by
// the host: calls of the single entry points from Python took twice its time.
// Scratch comes from the caller's workspace; nothing is kept between calls.
#include "fp8.cuh"

using namespace sffn;

namespace {

// The workspace in pieces of whole 256 bytes; with no base it only counts.
struct Scratch {
    char* base;
    size_t used = 0;
    void* take(size_t bytes) {
        void* p = base ? base + used : nullptr;
        used += (bytes + 255) & ~size_t(255);
        return p;
    }
};

long long up8(long long n) { return (n + 7) / 8 * 8; }
long long up16(long long n) { return (n + 15) / 16 * 16; }

// A 16-bit matrix; `odd`: its rows are copied to rows on 16 bytes.
struct Mat {
    const void* p;
    long long ld, rows, cols;
    bool odd;
};
Mat mat(const void* p, long long ld, long long rows, long long cols, bool odd) {
    return {p, rows == 1 && !odd ? up8(cols) : ld, rows, cols, odd};
}

struct Pads {
    int64_t desc[24];
    int count = 0;
    // The matrix as TMA reads it: itself, or its copy's place.
    void place(Mat& m, Scratch& ws) {
        if (!m.odd) return;
        void* to = ws.take((size_t)m.rows * up8(m.cols) * 2);
        const int64_t d[6] = {(int64_t)reinterpret_cast<intptr_t>(m.p), m.rows, m.cols, m.ld, (int64_t)reinterpret_cast<intptr_t>(to), up8(m.cols)};
        for (int i = 0; i < 6; ++i) desc[6 * count + i] = d[i];
        ++count;
        m.p = to, m.ld = up8(m.cols);
    }
    int run(void* stream) const { return count ? sffn_pad_rows16(count, desc, stream) : SFFN_OK; }
};

#define TRY(call)                 \
    do {                          \
        if (int _rc = (call)) return _rc; \
    } while (0)

// Rows that the few-row kernels take: up to 16 of any alignment, up to 64 where the
// weights' rows are on 16 bytes.  The 256-row tiles against them, us in bfloat16:
// gated 4096 x 14336, 16 rows 87 and 63, 17 rows 87 and 69, 64 rows 91 and 73; gated
// 2048 x 8192, 17 rows 34 and 29, 64 rows 35 and 35; gated 768 x 2048, 17 rows 20 and 15,
// 64 rows 23 and 24; y = x W^T with 14336 x 4096, 17 rows 28 and 27, 64 rows 28 and 27.
// They lose where tiles are few and K is long: 2048 x 8192, 17 rows 12.7 and 13.4; 1024 x
// 16384, 17 rows 14.0 and 16.5, 64 rows 15.6 and 18.1, the worst of the 13 shapes timed.
bool few_rows(long long T, int odd) { return T <= 16 || (T <= 64 && !odd); }

struct Product {
    int dtype;
    Scratch* ws;
    uint32_t* status;
    void* stream;
    bool count;  // sizes only
    // out [M, N] = A B^T (+ A2 B2^T)
    int operator()(void* out, long long ldo, long long M, long long N, long long K, const Mat& A, int a_mn, const Mat& B,
                   int b_mn, const Mat* A2 = nullptr, const Mat* B2 = nullptr, long long K2 = 0) const {
        const size_t before = ws->used, bytes = sffn_gemm16_workspace_bytes(M, N, K, K2);
        void* parts = bytes ? ws->take(bytes) : nullptr;
        if (count) return SFFN_OK;
        const int rc = sffn_gemm16(dtype, A.p, A.ld, a_mn, B.p, B.ld, b_mn, A2 ? A2->p : nullptr, A2 ? A2->ld : 0,
                                   B2 ? B2->p : nullptr, B2 ? B2->ld : 0, K2, M, N, K, out, ldo, parts, bytes, status, stream);
        ws->used = before;  // the next product's, on the same stream, may have the place
        return rc;
    }
};

bool dtype16(int d) { return d == SFFN_BF16 || d == SFFN_F16; }

// odd: bit 0 x, 1 W
int linear_fwd(int dtype, const void* x, long long ldx, const void* W, long long ldw, int odd, long long T, long long N,
               long long K, void* y, void* values, void* scales, Scratch& ws, uint32_t* status, void* stream, bool count) {
    Mat X = mat(x, ldx, T, K, odd & 1), V = mat(W, ldw, N, K, odd & 2);
    Pads pads;
    if (few_rows(T, odd & 2)) {
        if (!(odd & 2)) pads.place(X, ws);  // few rows are copied for the fast way through many
        if (count) return SFFN_OK;
        TRY(pads.run(stream));
        TRY(sffn_few_rows_mm(dtype, X.p, X.ld, V.p, V.ld, T, N, K, y, N, status, stream));
    } else {
        pads.place(X, ws);
        pads.place(V, ws);
        if (!count) TRY(pads.run(stream));
        TRY((Product{dtype, &ws, status, stream, count}(y, N, T, N, K, X, 0, V, 0)));
    }
    if (values && !count) TRY(sffn_fp8_pack(X.p, dtype, T, K, X.ld, values, up16(K), scales, stream));
    return SFFN_OK;
}

// odd: bit 0 dy, 1 W
int linear_bwd(int dtype, const void* dy, long long lddy, const void* W, long long ldw, int odd, const void* values,
               long long ldv, const void* scales, long long T, long long N, long long K, void* dx, void* dW, Scratch& ws,
               uint32_t* status, void* stream, bool count, bool want_x, bool want_W) {
    Mat DY = mat(dy, lddy, T, N, odd & 1), V = mat(W, ldw, N, K, odd & 2);
    const Product product{dtype, &ws, status, stream, count};
    Pads pads;
    pads.place(DY, ws);
    if (want_x) pads.place(V, ws);
    if (!count) TRY(pads.run(stream));
    if (want_W) {
        const size_t before = ws.used;
        const Mat kept = mat(ws.take((size_t)T * up8(K) * 2), up8(K), T, K, false);
        if (!count) TRY(sffn_fp8_unpack(values, ldv, scales, T, K, dtype, const_cast<void*>(kept.p), kept.ld, stream));
        TRY(product(dW, K, N, K, T, DY, 1, kept, 1));
        if (!count) ws.used = before;
    }
    if (want_x) TRY(product(dx, K, T, K, N, DY, 0, V, 1));
    return SFFN_OK;
}

// odd: bit 0 x, 1 Wg, 2 Wu, 3 W2
int gated_fwd(int dtype, int act, int keep, const void* x, long long ldx, const void* wg, long long ldg, const void* wu,
              long long ldu, const void* w2, long long ld2, int odd, long long T, long long D, long long F, void* y, void* g,
              void* u, void* gs, void* us, void* xv, void* xs, Scratch& ws, uint32_t* status, void* stream, bool count) {
    Mat X = mat(x, ldx, T, D, odd & 1), G = mat(wg, ldg, F, D, odd & 2), U = mat(wu, ldu, F, D, odd & 4),
        W2 = mat(w2, ld2, D, F, odd & 8);
    void* h = ws.take((size_t)T * up8(F) * 2);
    const Mat H = mat(h, up8(F), T, F, false);
    Pads pads;
    if (keep == SFFN_KEEP_NONE && few_rows(T, odd & 14)) {
        if (!(odd & 6)) pads.place(X, ws);  // few rows are copied for the fast way through many
        if (count) return SFFN_OK;
        TRY(pads.run(stream));
        return sffn_few_rows_ffn(dtype, act, X.p, X.ld, G.p, G.ld, U.p, U.ld, W2.p, W2.ld, T, D, F, h, H.ld, y, D, status, stream);
    }
    pads.place(X, ws);
    pads.place(G, ws);
    pads.place(U, ws);
    const bool few_down = few_rows(T, odd & 8);
    if (!few_down) pads.place(W2, ws);
    if (!count) {
        TRY(pads.run(stream));
        TRY(sffn_glu_up(dtype, act, X.p, X.ld, G.p, G.ld, U.p, U.ld, T, D, F, h, H.ld, keep, g, u,
                        keep == SFFN_KEEP_8 ? up16(F) : up8(F), gs, us, status, stream));
    }
    if (!few_down) TRY((Product{dtype, &ws, status, stream, count}(y, D, T, D, F, H, 0, W2, 0)));
    else if (!count) TRY(sffn_few_rows_mm(dtype, h, H.ld, W2.p, W2.ld, T, D, F, y, D, status, stream));
    if (keep == SFFN_KEEP_8 && !count) TRY(sffn_fp8_pack(X.p, dtype, T, D, X.ld, xv, up16(D), xs, stream));
    return SFFN_OK;
}

bool adjacent(const void* dwg, const void* dwu, long long D, long long F) {
    return dwu == static_cast<const char*>(dwg) + up8(F) * D * 2;
}
// Whether dWg and dWu are one product, which writes the rows between and behind them
// too: on request, and where there are none.  (By the two places alone it overwrote what
// lay there when separate buffers happened to be so far apart.)
bool joint_weights(int steps, const void* dwg, const void* dwu, long long D, long long F) {
    if (steps & (SFFN_GATED_JOINT | SFFN_GATED_APART)) return steps & SFFN_GATED_JOINT;
    return F % 8 == 0 && adjacent(dwg, dwu, D, F);
}

// odd: bit 0 dy, 1 Wg, 2 Wu, 3 W2, 4 x.  steps: SFFN_GATED_*, each on the same workspace.
int gated_bwd(int dtype, int act, int keep, int steps, const void* dy, long long lddy, const void* x, long long ldx,
              const void* wg, long long ldg, const void* wu, long long ldu, const void* w2, long long ld2, int odd,
              const void* g, const void* u, const void* gs, const void* us, const void* xv, const void* xs, long long T,
              long long D, long long F, void* dx, void* dwg, void* dwu, void* dw2, int want, Scratch& ws, uint32_t* status,
              void* stream, bool count) {
    const bool want_x = want & 1, want_g = want & 2, want_u = want & 4, want_2 = want & 8;
    const long long ldf = up8(F);
    Mat DY = mat(dy, lddy, T, D, odd & 1), G = mat(wg, ldg, F, D, odd & 2), U = mat(wu, ldu, F, D, odd & 4),
        W2 = mat(w2, ld2, D, F, odd & 8), X = mat(x, ldx, T, D, odd & 16);
    const Product product{dtype, &ws, status, stream, count};
    // places, the same ones at every step
    char* d = static_cast<char*>(ws.take((size_t)T * 2 * ldf * 2));  // dg | du a row, so that dWg and dWu may be one product
    const Mat H = mat(ws.take((size_t)T * ldf * 2), ldf, T, F, false);
    const Mat DG{d, 2 * ldf, T, F, false}, DU{d ? d + 2 * ldf : nullptr, 2 * ldf, T, F, false};
    Pads pads, pad_x;
    pads.place(DY, ws);
    pads.place(W2, ws);
    if (want_x) {
        pads.place(G, ws);
        pads.place(U, ws);
    }
    if (want_g || want_u) {
        if (keep == SFFN_KEEP_8) X = mat(ws.take((size_t)T * up8(D) * 2), up8(D), T, D, false);
        else pad_x.place(X, ws);
    }
    if ((steps & SFFN_GATED_DGRAD) && !count) {
        TRY(pads.run(stream));
        TRY(sffn_glu_dgrad(dtype, act, DY.p, DY.ld, W2.p, W2.ld, T, D, F, keep, g, u, keep == SFFN_KEEP_8 ? up16(F) : ldf, gs,
                           us, d, d + 2 * ldf, 2 * ldf, const_cast<void*>(H.p), ldf, status, stream));
    }
    if ((steps & SFFN_GATED_DW2) && want_2) TRY(product(dw2, F, D, F, T, DY, 1, H, 1));
    if ((steps & SFFN_GATED_DWGU) && (want_g || want_u)) {
        if (!count) {
            if (keep == SFFN_KEEP_8) TRY(sffn_fp8_unpack(xv, up16(D), xs, T, D, dtype, const_cast<void*>(X.p), X.ld, stream));
            else TRY(pad_x.run(stream));
        }
        const bool joint = want_g && want_u && joint_weights(steps, dwg, dwu, D, F);
        if (joint || (count && want_g && want_u)) {
            const Mat both{d, 2 * ldf, T, 2 * ldf, false};
            TRY(product(dwg, D, 2 * ldf, D, T, both, 1, X, 1));
        }
        if (!joint || count) {
            if (want_g) TRY(product(dwg, D, F, D, T, DG, 1, X, 1));
            if (want_u) TRY(product(dwu, D, F, D, T, DU, 1, X, 1));
        }
    }
    if ((steps & SFFN_GATED_DX) && want_x) TRY(product(dx, D, T, D, F, DG, 0, G, 1, &DU, &U, F));
    return SFFN_OK;
}

bool sizes_fit(long long T, long long D, long long F) {
    return T > 0 && D > 0 && F > 0 && T <= 0x7FFFFF00 && D <= 0x7FFFFF00 && F <= 0x3FFFFF00;
}

int enter(DeviceScope& scope, int dtype, const void* p, long long T, long long D, long long F, const void* ws, size_t have,
          size_t need, const void* status) {
    if (!dtype16(dtype)) return SFFN_ERR_DTYPE;
    if (!sizes_fit(T, D, F)) return SFFN_ERR_ARG;
    if (!p || !status) return SFFN_ERR_ARG;
    if (need && (!ws || have < need)) return SFFN_ERR_WORKSPACE;
    if (!aligned16(ws)) return SFFN_ERR_ALIGN;
    return scope.bind(p);
}

}  // namespace

extern "C" size_t sffn_ckpt_linear_workspace_bytes(int backward, int odd, int want, int64_t T, int64_t N, int64_t K) {
    if (!sizes_fit(T, N, K)) return 0;
    Scratch ws{nullptr};
    if (backward)
        linear_bwd(SFFN_BF16, nullptr, 0, nullptr, 0, odd, nullptr, 0, nullptr, T, N, K, nullptr, nullptr, ws, nullptr, nullptr, true,
                   want & 1, want & 2);
    else
        linear_fwd(SFFN_BF16, nullptr, 0, nullptr, 0, odd, T, N, K, nullptr, nullptr, nullptr, ws, nullptr, nullptr, true);
    return ws.used;
}

extern "C" int sffn_ckpt_linear(int dtype, const void* x, int64_t ldx, const void* W, int64_t ldw, int odd, int64_t T, int64_t N,
                                int64_t K, void* y, void* values, void* scales, void* workspace, size_t workspace_bytes,
                                uint32_t* status_dev, void* stream) {
    DeviceScope scope;
    TRY(enter(scope, dtype, x, T, N, K, workspace, workspace_bytes, sffn_ckpt_linear_workspace_bytes(0, odd, 0, T, N, K), status_dev));
    if (!W || !y || (values && !scales)) return SFFN_ERR_ARG;
    OuterScope outer(scope);
    Scratch ws{static_cast<char*>(workspace)};
    return linear_fwd(dtype, x, ldx, W, ldw, odd, T, N, K, y, values, scales, ws, status_dev, stream, false);
}

extern "C" int sffn_ckpt_linear_bwd(int dtype, const void* dy, int64_t lddy, const void* W, int64_t ldw, int odd,
                                    const void* values, int64_t ldv, const void* scales, int64_t T, int64_t N, int64_t K, void* dx,
                                    void* dW, void* workspace, size_t workspace_bytes, uint32_t* status_dev, void* stream) {
    DeviceScope scope;
    TRY(enter(scope, dtype, dy, T, N, K, workspace, workspace_bytes,
              sffn_ckpt_linear_workspace_bytes(1, odd, (dx ? 1 : 0) | (dW ? 2 : 0), T, N, K), status_dev));
    if ((dx && !W) || (dW && (!values || !scales))) return SFFN_ERR_ARG;
    OuterScope outer(scope);
    Scratch ws{static_cast<char*>(workspace)};
    return linear_bwd(dtype, dy, lddy, W, ldw, odd, values, ldv, scales, T, N, K, dx, dW, ws, status_dev, stream, false, dx != nullptr,
                      dW != nullptr);
}

extern "C" size_t sffn_fp8_linear_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    if (!sizes_fit(M, K, N)) return 0;
    Scratch ws{nullptr};
    ws.take((size_t)M * up16(K));
    ws.take((size_t)((M + 127) / 128 * fp8_block_tiles(K) * 512));
    if (!few_rows(M, 0)) ws.take(sffn_fp8_mm_workspace_bytes(M, N, K));
    return ws.used;
}

extern "C" int sffn_fp8_linear(const void* x, int dtype, int64_t ldx, const void* b, int64_t ldb, const void* b_scales, int64_t M,
                               int64_t N, int64_t K, void* C, int c_dtype, int64_t ldc, void* workspace, size_t workspace_bytes,
                               uint32_t* status_dev, void* stream) {
    if (!dtype_ok(dtype)) return SFFN_ERR_DTYPE;
    if (!sizes_fit(M, K, N) || !x) return SFFN_ERR_ARG;
    if (!workspace || workspace_bytes < sffn_fp8_linear_workspace_bytes(M, N, K)) return SFFN_ERR_WORKSPACE;
    if (!aligned16(workspace)) return SFFN_ERR_ALIGN;
    DeviceScope scope;
    TRY(scope.bind(x));
    OuterScope outer(scope);
    Scratch ws{static_cast<char*>(workspace)};
    void* values = ws.take((size_t)M * up16(K));
    void* scales = ws.take((size_t)((M + 127) / 128 * fp8_block_tiles(K) * 512));
    TRY(sffn_fp8_pack(x, dtype, M, K, ldx, values, up16(K), scales, stream));
    if (few_rows(M, 0))
        return few_rows_fp8(values, up16(K), scales, b, ldb, b_scales, M, N, K, C, c_dtype, ldc, true, status_dev, stream);
    const size_t bytes = sffn_fp8_mm_workspace_bytes(M, N, K);
    void* parts = bytes ? ws.take(bytes) : nullptr;
    return sffn_fp8_mm(values, up16(K), scales, b, ldb, b_scales, M, N, K, C, c_dtype, ldc, parts, bytes, status_dev, stream);
}

extern "C" size_t sffn_gated_ffn_workspace_bytes(int backward, int keep, int odd, int want, int64_t T, int64_t D, int64_t F) {
    if (!sizes_fit(T, D, F)) return 0;
    Scratch ws{nullptr};
    if (backward) {
        // parts of the products follow each other's places: the largest counts
        size_t most = 0;
        for (int step = 1; step <= 8; step *= 2) {
            Scratch one{nullptr};
            gated_bwd(SFFN_BF16, 0, keep, step, nullptr, 0, nullptr, 0, nullptr, 0, nullptr, 0, nullptr, 0, odd, nullptr, nullptr,
                      nullptr, nullptr, nullptr, nullptr, T, D, F, nullptr, nullptr, nullptr, nullptr, want, one, nullptr, nullptr, true);
            most = one.used > most ? one.used : most;
        }
        return most;
    }
    gated_fwd(SFFN_BF16, 0, keep, nullptr, 0, nullptr, 0, nullptr, 0, nullptr, 0, odd, T, D, F, nullptr, nullptr, nullptr, nullptr,
              nullptr, nullptr, nullptr, ws, nullptr, nullptr, true);
    return ws.used;
}

extern "C" int sffn_gated_ffn(int dtype, int act, int keep, const void* x, int64_t ldx, const void* wg, int64_t ldwg,
                              const void* wu, int64_t ldwu, const void* w2, int64_t ldw2, int odd, int64_t T, int64_t D, int64_t F,
                              void* y, void* g, void* u, void* g_scales, void* u_scales, void* x_values, void* x_scales,
                              void* workspace, size_t workspace_bytes, uint32_t* status_dev, void* stream) {
    DeviceScope scope;
    if (keep < SFFN_KEEP_NONE || keep > SFFN_KEEP_8) return SFFN_ERR_ARG;
    TRY(enter(scope, dtype, x, T, D, F, workspace, workspace_bytes, sffn_gated_ffn_workspace_bytes(0, keep, odd, 0, T, D, F), status_dev));
    if (!wg || !wu || !w2 || !y || (keep == SFFN_KEEP_8 && (!x_values || !x_scales))) return SFFN_ERR_ARG;
    OuterScope outer(scope);
    Scratch ws{static_cast<char*>(workspace)};
    return gated_fwd(dtype, act, keep, x, ldx, wg, ldwg, wu, ldwu, w2, ldw2, odd, T, D, F, y, g, u, g_scales, u_scales, x_values,
                     x_scales, ws, status_dev, stream, false);
}

extern "C" int sffn_gated_ffn_bwd(int dtype, int act, int keep, int steps, const void* dy, int64_t lddy, const void* x, int64_t ldx,
                                  const void* wg, int64_t ldwg, const void* wu, int64_t ldwu, const void* w2, int64_t ldw2, int odd,
                                  const void* g, const void* u, const void* g_scales, const void* u_scales, const void* x_values,
                                  const void* x_scales, int64_t T, int64_t D, int64_t F, void* dx, void* dwg, void* dwu, void* dw2,
                                  void* workspace, size_t workspace_bytes, uint32_t* status_dev, void* stream) {
    DeviceScope scope;
    if (keep != SFFN_KEEP_16 && keep != SFFN_KEEP_8) return SFFN_ERR_ARG;
    const int want = (dx ? 1 : 0) | (dwg ? 2 : 0) | (dwu ? 4 : 0) | (dw2 ? 8 : 0);
    TRY(enter(scope, dtype, dy, T, D, F, workspace, workspace_bytes, sffn_gated_ffn_workspace_bytes(1, keep, odd, want, T, D, F), status_dev));
    if ((steps & SFFN_GATED_JOINT) && ((steps & SFFN_GATED_APART) || !dwg || !dwu || !adjacent(dwg, dwu, D, F))) return SFFN_ERR_ARG;
    if (!wg || !wu || !w2 || ((dwg || dwu) && (keep == SFFN_KEEP_8 ? !x_values || !x_scales : !x))) return SFFN_ERR_ARG;
    OuterScope outer(scope);
    Scratch ws{static_cast<char*>(workspace)};
    return gated_bwd(dtype, act, keep, steps, dy, lddy, x, ldx, wg, ldwg, wu, ldwu, w2, ldw2, odd, g, u, g_scales, u_scales, x_values,
                     x_scales, T, D, F, dx, dwg, dwu, dw2, want, ws, status_dev, stream, false);
}
