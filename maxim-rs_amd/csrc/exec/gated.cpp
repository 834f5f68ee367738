// The gated Dense's host side (include/maxim_block_ops.h): argument checks and the
// launches. Forward it is a product of ops.cpp with pairs of lines, backward a
// pass that forms dz and a Dense's two products.

#include "maxim_block_ops.h"
#include "ops_host.hpp"

namespace mxops {

// x, y and z in the results' order, the weights either way. An axis of one
// element has no stride of its own: the order that the call has is said.
static Product gated_product(const mxh_mat &x, const mxh_mat &w, const mxh_mat &y, bool by_cols) {
    Product p;
    p.dtype = y.dtype;
    p.k = x.cols;
    p.c = y.data;
    const Operand weights = along_cols(w) ? Operand{w.data, w.row_stride, 1, false, 'k'}
                                          : Operand{w.data, 1, w.col_stride, false, 'm'};
    if (by_cols) {
        p.pair = Pair::kN;
        p.m = y.rows, p.n = y.cols, p.ldc = y.row_stride;
        p.a = Operand{x.data, x.row_stride, 1, false, 'k'};
        p.b = weights;
    } else {
        p.pair = Pair::kM;
        p.m = y.cols, p.n = y.rows, p.ldc = y.col_stride;
        p.a = weights;
        p.b = Operand{x.data, 1, x.col_stride, false, 'm'};
    }
    return p;
}

static int64_t halves(const mxh_mat &w) {
    if (w.rows % 2) throw Error("w: " + std::to_string(w.rows) + " rows are no gate's and as many values'");
    return w.rows / 2;
}

// The operands' sizes, types and strides, and the order that they have.
static bool check_gated(const mxh_mat *x, const mxh_mat *w, const mxh_mat *y, const mxh_mat *z) {
    const mxh_mat &X = need(x, "x"), &W = need(w, "w"), &Y = need(y, "y");
    check_first(X, "x");
    check_mat(W, "w", X.dtype, W.rows, X.cols);
    check_mat(Y, "y", X.dtype, X.rows, halves(W));
    check_out(Y, "y");
    if (z) {
        check_mat(*z, "z", x->dtype, x->rows, w->rows);
        check_out(*z, "z");
    }
    return common_order({x}, {y, z});
}

static mxh_mat like(const mxh_mat &m, int64_t cols) {
    mxh_mat r = m;
    r.cols = cols;
    return r;
}

// The dz pass's blocks along the rows. In planar order a block's run is whole
// turns of its 256 threads' vectors, as many as leave about 2048 blocks (64
// bf16 features of 71680 positions: in 32 runs of 1.1 turns 15.9 us, in 35 of one
// 14.4).
static int64_t gated_parts(const mxh_mat &dy, bool by_cols) {
    if (by_cols || !dy.cols || !dy.rows) return dz_parts(dy, by_cols);
    const int64_t turn = 256 * 16 / (int64_t)type_size(dy.dtype), want = cdiv(2048, dy.cols);
    return std::min<int64_t>(65535, cdiv(dy.rows, turn * std::max<int64_t>(1, dy.rows / (turn * want))));
}

// The dz pass's blocks across the features.
static int64_t gated_across(const mxh_mat &dy, bool by_cols) {
    return by_cols ? cdiv(dy.cols, 64 * 16 / (int64_t)type_size(dy.dtype)) : dy.cols;
}
// So many blocks' largest magnitudes each block reads for itself (16 KiB, from
// L2); more of them one block reads for all.
constexpr int64_t kFewTops = 4096;
// Blocks that form dz again, which mostly leave at once (4096 x 2 x 2048 out of
// range: 256 and 512 take 4 us more, 2048 nothing less).
constexpr int64_t kBlocksAgain = 1024;

static BwdLayout gated_layout(const mxh_mat &dy, bool by_cols, const mxh_mat &x, const mxh_mat &w, const mxh_mat *dx,
                              const mxh_mat *dw, const mxh_vec *db) {
    BwdLayout l;
    l.dz = like(dy, 2 * dy.cols);
    if (dx || dw) place_dz(l, dy, 2 * dy.cols, by_cols);
    if (db) {
        l.parts = gated_parts(dy, by_cols);
        l.part_bytes = up((uint64_t)l.parts * 2 * dy.cols * 4);
    }
    // fp16: a magnitude a block, the largest, and what the products take back
    if (l.dz_bytes && dy.dtype == MXH_F16)
        l.top_bytes = up((uint64_t)(gated_across(dy, by_cols) * gated_parts(dy, by_cols) + 2) * 4);
    if (dx && !empty(*dx)) l.product_bytes = std::max(l.product_bytes, plan_of(product_dx(l, w, *dx)).bytes);
    if (dw && !empty(*dw)) l.product_bytes = std::max(l.product_bytes, plan_of(product_dw(l, x, *dw)).bytes);
    return l;
}

}  // namespace mxops

using namespace mxops;

extern "C" {

int mxh_gated_workspace(const mxh_mat *x, const mxh_mat *w, const mxh_mat *y, const mxh_mat *z, uint64_t *bytes) {
    return guard([&] {
        if (!bytes) throw Error("bytes: missing");
        *bytes = 0;
        const bool by_cols = check_gated(x, w, y, z);
        if (!empty(*y)) *bytes = plan_of(gated_product(*x, *w, *y, by_cols)).bytes;
    });
}

int mxh_gated(int device, void *stream, const mxh_mat *x, const mxh_mat *w, const mxh_vec *bias, int act, float slope,
              const mxh_mat *y, const mxh_mat *z, void *workspace, uint64_t workspace_bytes) {
    return guard([&] {
        const bool by_cols = check_gated(x, w, y, z);
        const mxh_mat &X = *x, &W = *w, &Y = *y;
        check_act(act);
        if (bias) check_vec(*bias, "bias", W.rows, X.dtype);
        for (const mxh_mat *o : {y, z}) {
            if (!o) continue;
            refuse_overlap(*o, "an output", X, "x");
            refuse_overlap(*o, "an output", W, "w");
            if (bias) refuse_overlap(*o, "an output", line(*bias), "bias");
        }
        if (z) refuse_overlap(Y, "y", *z, "z");
        if (empty(Y)) return;
        Product p = gated_product(X, W, Y, by_cols);
        check_workspace(workspace, workspace_bytes, plan_of(p).bytes);
        p.bias = bias;
        p.bias_rows = !by_cols;
        p.act = act;
        p.slope = slope;
        if (z) p.z = z->data, p.ldz = by_cols ? z->row_stride : z->col_stride;
        Launches launches;
        product(launches, p, workspace);
        launches.run(device, stream);
    });
}

int mxh_gated_backward_workspace(const mxh_mat *dy, const mxh_mat *x, const mxh_mat *w, const mxh_mat *dx,
                                 const mxh_mat *dw, const mxh_vec *db, uint64_t *bytes) {
    return guard([&] {
        if (!bytes) throw Error("bytes: missing");
        const mxh_mat &X = need(x, "x"), &W = need(w, "w"), &DY = need(dy, "dy");
        check_first(X, "x");
        check_mat(W, "w", X.dtype, W.rows, X.cols);
        check_mat(DY, "dy", X.dtype, X.rows, halves(W));
        if (dx) check_mat(*dx, "dx", x->dtype, x->rows, x->cols);
        if (dw) check_mat(*dw, "dw", x->dtype, w->rows, w->cols);
        *bytes = std::max(gated_layout(*dy, true, *x, *w, dx, dw, db).total(),
                          gated_layout(*dy, false, *x, *w, dx, dw, db).total());
    });
}

int mxh_gated_backward(int device, void *stream, const mxh_mat *dy, const mxh_mat *x, const mxh_mat *w,
                       const mxh_mat *z, int act, float slope, const mxh_mat *dx, const mxh_mat *dw,
                       const mxh_vec *db, void *workspace, uint64_t workspace_bytes) {
    return guard([&] {
        const mxh_mat &X = need(x, "x"), &W = need(w, "w"), &DY = need(dy, "dy"), &Z = need(z, "z");
        check_first(X, "x");
        check_mat(W, "w", X.dtype, W.rows, X.cols);
        check_mat(DY, "dy", X.dtype, X.rows, halves(W));
        check_mat(Z, "z", X.dtype, X.rows, W.rows);
        check_act(act);
        if (dx) {
            check_mat(*dx, "dx", X.dtype, X.rows, X.cols);
            check_out(*dx, "dx");
        }
        if (dw) {
            check_mat(*dw, "dw", X.dtype, W.rows, W.cols);
            check_out(*dw, "dw");
        }
        if (db) check_vec(*db, "db", W.rows, X.dtype);
        const bool by_cols = common_order({dy, z}, {});
        const mxh_mat dbl = db ? line(*db) : mxh_mat{};
        const mxh_mat *outs[] = {dx, dw, db ? &dbl : nullptr}, *ins[] = {dy, x, w, z};
        const char *on_[] = {"dx", "dw", "db"}, *in_[] = {"dy", "x", "w", "z"};
        for (int i = 0; i < 3; ++i) {
            if (!outs[i]) continue;
            for (int j = 0; j < 4; ++j) refuse_overlap(*outs[i], on_[i], *ins[j], in_[j]);
            for (int j = 0; j < i; ++j)
                if (outs[j]) refuse_overlap(*outs[i], on_[i], *outs[j], on_[j]);
        }
        BwdLayout l = gated_layout(DY, by_cols, X, W, dx, dw, db);
        check_workspace(workspace, workspace_bytes, l.total());
        Launches launches;
        char *ws = static_cast<char *>(workspace);
        const std::string t = kTypeName[X.dtype];
        OpsGatedDzArgs dz{};
        OpsDzArgs &a = dz.d;
        a.dy = DY.data;
        a.z = Z.data;
        a.rows = DY.rows;
        a.cols = DY.cols;
        a.dyrs = DY.row_stride, a.dycs = DY.col_stride;
        a.zrs = Z.row_stride, a.zcs = Z.col_stride;
        if (l.dz_bytes) l.dz.data = a.dz = ws, a.drs = l.dz.row_stride, a.dcs = l.dz.col_stride;
        // one part, with rows: its sums are db itself
        const bool whole = db && l.parts == 1 && DY.rows;
        if (whole) dz.db = db->data, dz.db_type = db->dtype;
        else if (db) a.part = reinterpret_cast<float *>(ws + l.dz_bytes);
        a.nparts = (int32_t)gated_parts(DY, by_cols);
        a.act = act;
        a.slope = slope;
        const float *back = nullptr;
        if ((a.dz || a.part || dz.db) && !empty(DY)) {
            const std::string name = (by_cols ? "mxg_dz_rows_" : "mxg_dz_planar_") + t;
            const int64_t across = gated_across(DY, by_cols), blocks = across * a.nparts;
            if (l.top_bytes) dz.top = reinterpret_cast<float *>(ws + l.dz_bytes + l.part_bytes);
            launches.add(name, across, a.nparts, 256, dz);
            if (l.top_bytes) {
                dz.ntop = (int32_t)blocks;
                back = dz.back = dz.top + blocks + 1;
                if (blocks > kFewTops) {
                    dz.pass = MXO_DZ_TOPS;
                    launches.add(name, 1, 1, 256, dz);
                    dz.top += blocks, dz.ntop = 1;
                }
                dz.pass = MXO_DZ_SCALED;
                launches.add(name, across, std::max<int64_t>(1, std::min<int64_t>(a.nparts, kBlocksAgain / across)), 256, dz);
            }
        }
        void *pw = ws + l.dz_bytes + l.part_bytes + l.top_bytes;
        auto gradient = [&](Product p, OpsGemmArgs *later) {
            p.back = back;
            product(launches, p, pw, later);
        };
        if (dx && !empty(*dx)) gradient(product_dx(l, W, *dx), nullptr);
        OpsGradJoinArgs j{};
        if (dw && !empty(*dw)) gradient(product_dw(l, X, *dw), db && !whole ? &j.g : nullptr);
        const int64_t parts = DY.rows ? l.parts : 0, quads = j.g.m * cdiv(j.g.n, 4);
        // dw's splits and the bias's parts in one launch, where dw is small
        if (j.g.splits > 1 && quads <= 65536) {
            j.part = a.part;
            j.out = db->data;
            j.n = (int32_t)W.rows;
            j.nparts = (int32_t)parts;
            j.first = (int32_t)cdiv(quads, 16);
            j.dtype = db->dtype;
            launches.add("mxg_grad_join_" + t, j.first + cdiv(W.rows, 4), 1, 256, j);
        } else {
            if (j.g.splits > 1) join_product(launches, j.g, X.dtype);
            if (db && !whole) join(launches, a.part, parts, W.rows, db->data, nullptr, db->dtype);
        }
        launches.run(device, stream);
    });
}

}  // extern "C"
