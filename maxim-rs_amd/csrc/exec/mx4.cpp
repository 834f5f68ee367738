// The 4-bit operators' host side (include/maxim_block_ops.h): argument checks,
// the choice of tile and split, and the launches.

#include "../ops/mx4_args.h"
#include "maxim_block_ops.h"
#include "ops_host.hpp"

namespace mxops {

// Lines of whole tiles, scales of whole groups.
static int64_t tiles_of(int64_t cols) { return cdiv(cols, 256); }
static uint64_t code_bytes(int64_t rows, int64_t cols) { return (uint64_t)rows * tiles_of(cols) * 128; }
static uint64_t scale_bytes(int64_t rows, int64_t cols) { return (uint64_t)cdiv(rows, 64) * tiles_of(cols) * 512; }

// A tile's lines are offsets of 31 bits: 256 of 2^23 bytes at most.
constexpr int64_t kMaxFeatures = (int64_t(1) << 24) - 256;

static void check_size(int64_t rows, int64_t cols, const char *what) {
    if (rows < 0 || cols < 0 || rows > kMaxExtent || cols > kMaxFeatures)
        throw Error(std::string(what) + ": [" + std::to_string(rows) + "][" + std::to_string(cols) + "] is out of range");
}

static mxh_mat bytes_of(const void *p, uint64_t n) { return line(p, (int64_t)(n / 4), MXH_F32); }

static void check_mx4(const mxh_mx4 *q, const char *what, int64_t rows, int64_t cols) {
    const std::string w = what;
    if (!q) throw Error(w + ": missing");
    check_size(q->rows, q->cols, what);
    if (q->rows != rows || q->cols != cols)
        throw Error(w + ": [" + std::to_string(q->rows) + "][" + std::to_string(q->cols) + "], expected [" +
                    std::to_string(rows) + "][" + std::to_string(cols) + "]");
    if (!rows || !cols) return;
    if (!q->codes || !q->scales) throw Error(w + ": no data");
    if ((uintptr_t)q->codes % 16 || (uintptr_t)q->scales % 16) throw Error(w + ": not aligned to 16 bytes");
}

static void code_launch(Launches &launches, const char *way, const mxh_mat &x, bool by_cols, void *codes, void *scales) {
    Mx4CodeArgs a{};
    a.x = a.y = x.data;
    a.codes = static_cast<uint8_t *>(codes);
    a.scales = static_cast<uint8_t *>(scales);
    a.rows = x.rows, a.cols = x.cols;
    // an axis of one element has no stride of its own
    a.rs = by_cols ? x.row_stride : 1, a.cs = by_cols ? 1 : x.col_stride;
    a.tiles = (int32_t)tiles_of(x.cols);
    // positions a block: rows are quantised by half groups, planes by 4 bytes a lane
    const int64_t at = by_cols ? (way[0] == 'q' ? 32 : 64) : 64 * 4 / (int64_t)type_size(x.dtype);
    launches.add(std::string("mxq_") + way + (by_cols ? "_rows_" : "_planar_") + kTypeName[x.dtype],
                 cdiv(x.rows, at) * a.tiles, 1, 256, a);
}

// What a tile costs in us, as kTiles16 of ops.cpp has it: a step is 128 bytes of
// a line, 256 elements; `rest` with the launch that quantises x. Measured on
// products of 16 to 4096 rows.
struct Cost {
    int b, stages, fit;
    double one, all, rest;
};
static const Cost kTilesMx4[] = {{256, 2, 1, 1.65, 1.65, 12.0}, {128, 2, 2, 1.0, 1.3, 8.0}, {64, 4, 2, 0.3, 0.45, 6.0}};

struct Mx4Plan {
    bool few = false;  // the kernel of few rows
    int b = 0, stages = 0;
    int64_t splits = 1, chunk = 0;
    uint64_t codes = 0, scales = 0, parts = 0;
    uint64_t bytes() const { return codes + scales + parts; }
};

// The tile and the cut of k that take the least time by those costs, or for up
// to 16 rows the kernel that quantises x as it reads it: a block for 16 columns
// and all of k, whose waves take an eighth of its tiles each, one after the
// other. bf16, one row and 16: k = 4096 to 4096 columns 6.4 and 9.0 us, as tiles
// of 64 9.2 and 9.5; k = 16384 to 1024 columns 15.9 and 22.7, tiles cut in eight
// 10.4 and 11.0. 1024 x 4096 x 4096: 128 x 128 24 us, 64 x 64 26, 256 x 256 37;
// 4096 x 256 x 4096: 20, 34 and 17.
static Mx4Plan mx4_plan(const mxh_mat &x, int64_t n, bool by_cols) {
    Mx4Plan p;
    const int64_t steps = std::max<int64_t>(1, tiles_of(x.cols));
    double least = std::numeric_limits<double>::infinity();
    for (const Cost &t : kTilesMx4) {
        const int64_t tiles = cdiv(x.rows, t.b) * cdiv(n, t.b);
        for (int64_t cut : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64}) {
            const int64_t each = cdiv(steps, cut), splits = cdiv(steps, each);
            if (cut > 1 && each < 2) continue;
            const int64_t total = tiles * splits, full = total / (256 * t.fit), left = cdiv(total % (256 * t.fit), 256);
            double us = full * (each * t.all + t.rest);
            if (left) us += each * std::max(t.one, t.all * left / t.fit) + t.rest;
            if (splits > 1) us += 3.0 + (double)splits * x.rows * n * 8 / 5e6;
            if (us >= least) continue;
            least = us;
            p.b = t.b, p.stages = t.stages, p.splits = splits, p.chunk = each;
        }
    }
    if (by_cols && x.rows <= 16 && along_cols(x)) {
        const double few = 3.3 + 0.065 * x.rows + (1.5 + 0.05 * x.rows) * cdiv(steps, 8) * std::max(1.0, cdiv(n, 16) / 256.0);
        if (few <= least) {
            p.few = true;
            return p;
        }
    }
    p.codes = up(code_bytes(x.rows, x.cols));
    p.scales = up(scale_bytes(x.rows, x.cols));
    p.parts = p.splits > 1 ? (uint64_t)p.splits * x.rows * n * 4 : 0;
    return p;
}

// The operands' sizes, types and strides, and the order that the results have.
static bool check_dense(const mxh_mat *x, const mxh_mx4 *w, const mxh_mat *residual, const mxh_mat *y) {
    const mxh_mat &X = need(x, "x"), &Y = need(y, "y");
    check_first(X, "x");
    if (!w) throw Error("w: missing");
    check_mx4(w, "w", w->rows, X.cols);
    check_mat(Y, "y", X.dtype, X.rows, w->rows);
    check_out(Y, "y");
    if (residual) check_mat(*residual, "residual", x->dtype, x->rows, w->rows);
    return common_order({residual}, {y});
}

}  // namespace mxops

using namespace mxops;

extern "C" {

int mxh_mx4_size(int64_t rows, int64_t cols, uint64_t *codes, uint64_t *scales) {
    return guard([&] {
        if (!codes || !scales) throw Error("codes, scales: missing");
        check_size(rows, cols, "the matrix");
        *codes = code_bytes(rows, cols);
        *scales = scale_bytes(rows, cols);
    });
}

int mxh_mx4_quantize(int device, void *stream, const mxh_mat *x, const mxh_mx4 *q) {
    return guard([&] {
        check_first(need(x, "x"), "x");
        check_mx4(q, "q", x->rows, x->cols);
        if (empty(*x)) return;
        const mxh_mat c = bytes_of(q->codes, code_bytes(x->rows, x->cols)), s = bytes_of(q->scales, scale_bytes(x->rows, x->cols));
        refuse_overlap(c, "codes", *x, "x");
        refuse_overlap(s, "scales", *x, "x");
        refuse_overlap(c, "codes", s, "scales");
        Launches launches;
        code_launch(launches, "quantize", *x, along_cols(*x), q->codes, q->scales);
        launches.run(device, stream);
    });
}

int mxh_mx4_dequantize(int device, void *stream, const mxh_mx4 *q, const mxh_mat *y) {
    return guard([&] {
        check_first(need(y, "y"), "y");
        check_out(*y, "y");
        check_mx4(q, "q", y->rows, y->cols);
        if (empty(*y)) return;
        refuse_overlap(*y, "y", bytes_of(q->codes, code_bytes(y->rows, y->cols)), "codes");
        refuse_overlap(*y, "y", bytes_of(q->scales, scale_bytes(y->rows, y->cols)), "scales");
        Launches launches;
        code_launch(launches, "dequantize", *y, out_by_cols(*y), q->codes, q->scales);
        launches.run(device, stream);
    });
}

int mxh_mx4_dense_workspace(const mxh_mat *x, const mxh_mx4 *w, const mxh_mat *residual, const mxh_mat *y,
                            uint64_t *bytes) {
    return guard([&] {
        if (!bytes) throw Error("bytes: missing");
        *bytes = 0;
        const bool by_cols = check_dense(x, w, residual, y);
        if (!empty(*y)) *bytes = mx4_plan(*x, w->rows, by_cols).bytes();
    });
}

int mxh_mx4_dense(int device, void *stream, const mxh_mat *x, const mxh_mx4 *w, const mxh_vec *bias, int act, float slope,
                  const mxh_mat *residual, const mxh_mat *y, void *workspace, uint64_t workspace_bytes) {
    return guard([&] {
        const bool by_cols = check_dense(x, w, residual, y);
        const mxh_mat &X = *x, &Y = *y;
        check_act(act);
        if (bias) check_vec(*bias, "bias", w->rows, X.dtype);
        refuse_overlap(Y, "y", X, "x");
        refuse_overlap(Y, "y", bytes_of(w->codes, code_bytes(w->rows, w->cols)), "w's codes");
        refuse_overlap(Y, "y", bytes_of(w->scales, scale_bytes(w->rows, w->cols)), "w's scales");
        if (bias) refuse_overlap(Y, "y", line(*bias), "bias");
        if (residual && !same(*residual, Y)) refuse_overlap(Y, "y", *residual, "the residual");
        if (empty(Y)) return;
        const Mx4Plan p = mx4_plan(X, w->rows, by_cols);
        check_workspace(workspace, workspace_bytes, p.bytes());
        Launches launches;
        uint8_t *ws = static_cast<uint8_t *>(workspace);
        const std::string t = kTypeName[X.dtype];
        Mx4GemmArgs m{};
        OpsGemmArgs &g = m.g;
        g.c = Y.data;
        g.m = (int32_t)(by_cols ? X.rows : w->rows);
        g.n = (int32_t)(by_cols ? w->rows : X.rows);
        g.k = (int32_t)tiles_of(X.cols);
        g.ldc = by_cols ? Y.row_stride : Y.col_stride;
        if (residual) g.res = residual->data, g.ldr = by_cols ? residual->row_stride : residual->col_stride;
        if (bias) {
            g.bias = bias->data;
            g.bias_f32 = bias->dtype == MXH_F32 && X.dtype != MXH_F32;
            g.bias_rows = !by_cols;
        }
        g.act = act;
        g.slope = slope;
        g.splits = (int32_t)p.splits;
        g.kchunk = (int32_t)p.chunk;
        const uint8_t *wc = static_cast<uint8_t *>(w->codes), *wsc = static_cast<uint8_t *>(w->scales);
        if (p.few) {
            m.a = static_cast<uint8_t *>(X.data), g.lda = X.row_stride, m.cols = X.cols;
            m.b = wc, m.sb = wsc;
            launches.add("mxq_skinny_" + t, cdiv(g.n, 16), 1, 512, m);
            launches.run(device, stream);
            return;
        }
        if (X.cols) code_launch(launches, "quantize", X, along_cols(X), ws, ws + p.codes);
        m.a = by_cols ? ws : wc, m.sa = by_cols ? ws + p.codes : wsc;
        m.b = by_cols ? wc : ws, m.sb = by_cols ? wsc : ws + p.codes;
        g.part = reinterpret_cast<float *>(ws + p.codes + p.scales);
        g.tiles_m = (int32_t)cdiv(g.m, p.b);
        g.tiles_n = (int32_t)cdiv(g.n, p.b);
        const std::string b = std::to_string(p.b);
        launches.add("mxq_gemm_" + t + "_" + b + "x" + b + "_d" + std::to_string(p.stages),
                     (int64_t)g.tiles_m * g.tiles_n * p.splits, 1, p.b == 256 ? 512 : 256, m);
        if (p.splits > 1) {
            const bool deep = p.splits >= 16;
            launches.add((deep ? "mxo_join8_" : "mxo_join_") + t,
                         std::min<int64_t>(4096, cdiv(g.m * cdiv(g.n, 4), deep ? 32 : 256)), 1, 256, g);
        }
        launches.run(device, stream);
    });
}

}  // extern "C"
