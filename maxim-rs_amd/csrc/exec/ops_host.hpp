// What the operators' host files share (include/maxim_ops.h): the kernels'
// loading and launching, the checks of operands, and the products of ops.cpp.
#pragma once

#include "maxim_ops.h"

#include <algorithm>
#include <array>
#include <cstring>
#include <iterator>
#include <limits>
#include <string>

#include "../ops/ops_args.h"
#include "hip_api.hpp"
#include "host.hpp"

namespace mxops {

using mx::Error;
using mxh::check;
using mxh::hip;

constexpr int kMaxDevices = 64;
constexpr int64_t kMaxExtent = std::numeric_limits<int32_t>::max() - 1024;

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ------------------------------------------------------------ the kernels

// The calling thread's current device, put back on the way out.
struct OnDevice {
    int before = -1;
    explicit OnDevice(int dev) {
        if (dev < 0 || dev >= kMaxDevices) throw Error("device ordinal out of range");
        int now = -1;
        check(hip().hipGetDevice(&now), "hipGetDevice");
        if (now != dev) {
            check(hip().hipSetDevice(dev), "hipSetDevice");
            before = now;
        }
    }
    ~OnDevice() {
        if (before >= 0) hip().hipSetDevice(before);
    }
    OnDevice(const OnDevice &) = delete;
    OnDevice &operator=(const OnDevice &) = delete;
};

// The kernel of this name, from the code object its prefix names, loaded on
// first use.
mxh::hipFunction_t function(int dev, const std::string &name);
// All of them.
void load_all(int dev);

// A call's launches, of which none is made before all are known to fit: the
// threads of a launch are counted in 32 bits.
class Launches {
    struct One {
        std::string name;
        unsigned gx, gy, block;
        alignas(8) char args[200];
    };
    // a gated Dense's backward pass: dz in up to three launches and its join, twice
    // packing, product and join
    static constexpr int kMost = 10;
    One at_[kMost];
    int n_ = 0;

public:
    template <typename A>
    void add(const std::string &name, int64_t gx, int64_t gy, unsigned block, const A &args) {
        static_assert(sizeof(A) <= sizeof(One::args), "");
        if (gx > (int64_t)UINT32_MAX / block || gy > 65535)
            throw Error("the operands are too large: " + name + " would take more threads than one launch can have");
        One &o = at_[n_++];
        o.name = name;
        o.gx = (unsigned)gx, o.gy = (unsigned)gy, o.block = block;
        std::memcpy(o.args, &args, sizeof(A));
    }
    void run(int dev, void *stream) {
        OnDevice on(dev);
        mxh::hipFunction_t f[kMost];
        for (int i = 0; i < n_; ++i) f[i] = function(dev, at_[i].name);
        for (int i = 0; i < n_; ++i) {
            One &o = at_[i];
            void *params[] = {o.args};
            check(hip().hipModuleLaunchKernel(f[i], o.gx, o.gy, 1, o.block, 1, 1, 0, (mxh::hipStream_t)stream, params,
                                              nullptr),
                  o.name.c_str());
        }
    }
};

// ------------------------------------------------------------- operands

inline const char *const kTypeName[] = {"f32", "f16", "bf16"};
inline size_t type_size(int t) { return t == MXH_F32 ? 4 : 2; }

inline std::string shape(const mxh_mat &m) { return "[" + std::to_string(m.rows) + "][" + std::to_string(m.cols) + "]"; }

inline bool empty(const mxh_mat &m) { return m.rows == 0 || m.cols == 0; }
// Contiguous along columns (features), or along rows (positions).
inline bool along_cols(const mxh_mat &m) { return m.col_stride == 1 || m.cols <= 1; }
inline bool along_rows(const mxh_mat &m) { return m.row_stride == 1 || m.rows <= 1; }

inline const mxh_mat &need(const mxh_mat *m, const char *what) {
    if (!m) throw Error(std::string(what) + ": missing");
    return *m;
}

inline void check_mat(const mxh_mat &m, const char *what, int dtype, int64_t rows, int64_t cols) {
    const std::string w = what;
    if (m.dtype < MXH_F32 || m.dtype > MXH_BF16) throw Error(w + ": unknown type " + std::to_string(m.dtype));
    if (m.dtype != dtype) throw Error(w + ": " + kTypeName[m.dtype] + " where x is " + kTypeName[dtype]);
    if (m.rows != rows || m.cols != cols)
        throw Error(w + ": " + shape(m) + ", expected [" + std::to_string(rows) + "][" + std::to_string(cols) + "]");
    if (m.rows < 0 || m.cols < 0 || m.rows > kMaxExtent || m.cols > kMaxExtent)
        throw Error(w + ": " + shape(m) + " is out of range");
    if (m.row_stride < 0 || m.col_stride < 0) throw Error(w + ": a negative stride");
    if (empty(m)) return;
    if (!m.data) throw Error(w + ": no data");
    if (!along_cols(m) && !along_rows(m))
        throw Error(w + ": neither rows nor columns are contiguous (strides " + std::to_string(m.row_stride) + ", " +
                    std::to_string(m.col_stride) + ")");
    if ((uintptr_t)m.data % type_size(m.dtype)) throw Error(w + ": not aligned to its element");
    // the farthest element's offset in bytes has to be a number
    const __int128 far = ((__int128)(m.rows - 1) * m.row_stride + (__int128)(m.cols - 1) * m.col_stride) * 4;
    if (far > std::numeric_limits<int64_t>::max() / 2) throw Error(w + ": strides out of range");
}

inline void check_first(const mxh_mat &x, const char *what) { check_mat(x, what, x.dtype, x.rows, x.cols); }

inline void check_vec(const mxh_vec &v, const char *what, int64_t n, int dtype) {
    const std::string w = what;
    if (v.n != n) throw Error(w + ": " + std::to_string(v.n) + " elements, expected " + std::to_string(n));
    if (v.dtype != MXH_F32 && v.dtype != dtype) throw Error(w + ": its type is neither fp32 nor x's");
    if (n && !v.data) throw Error(w + ": no data");
    if ((uintptr_t)v.data % type_size(v.dtype)) throw Error(w + ": not aligned to its element");
}

// The memory order that all of a call's matrices have: true, features
// contiguous; false, positions. (One of a single row or column has both.)
inline bool out_by_cols(const mxh_mat &m) { return along_cols(m) && (m.rows <= 1 || m.row_stride >= m.cols); }
inline bool out_by_rows(const mxh_mat &m) { return along_rows(m) && (m.cols <= 1 || m.col_stride >= m.rows); }
inline bool common_order(std::initializer_list<const mxh_mat *> ins, std::initializer_list<const mxh_mat *> outs) {
    bool cols = true, rows = true;
    for (const mxh_mat *m : ins)
        if (m && !empty(*m)) cols = cols && along_cols(*m), rows = rows && along_rows(*m);
    for (const mxh_mat *m : outs)
        if (m && !empty(*m)) cols = cols && out_by_cols(*m), rows = rows && out_by_rows(*m);
    if (!cols && !rows) throw Error("the matrices differ in memory order");
    return cols;
}

// Elements of an output may not share storage.
inline void check_out(const mxh_mat &m, const char *what) {
    if (empty(m)) return;
    if (!out_by_cols(m) && !out_by_rows(m)) throw Error(std::string(what) + ": elements of an output share storage");
}

struct Range {
    uintptr_t lo, hi;
};
inline Range range(const mxh_mat &m) {
    const uintptr_t p = (uintptr_t)m.data;
    const uint64_t far = (uint64_t)(m.rows - 1) * m.row_stride + (uint64_t)(m.cols - 1) * m.col_stride + 1;
    return {p, p + far * type_size(m.dtype)};
}
inline bool apart(Range a, Range b) { return a.hi <= b.lo || b.hi <= a.lo; }

// Whether two views share an element: by their ranges, and where these cross
// and the strides agree (slices of one buffer), by their offset in it.
inline bool overlap(const mxh_mat &a, const mxh_mat &b) {
    if (empty(a) || empty(b) || apart(range(a), range(b))) return false;
    if (a.dtype != b.dtype) return true;
    int64_t ld, inner_a, inner_b, outer_a, outer_b;
    if (along_cols(a) && along_cols(b) && a.row_stride == b.row_stride) {
        ld = a.row_stride, inner_a = a.cols, inner_b = b.cols, outer_a = a.rows, outer_b = b.rows;
    } else if (along_rows(a) && along_rows(b) && a.col_stride == b.col_stride) {
        ld = a.col_stride, inner_a = a.rows, inner_b = b.rows, outer_a = a.cols, outer_b = b.cols;
    } else {
        return true;
    }
    const int64_t size = (int64_t)type_size(a.dtype);
    const int64_t bytes = (int64_t)((uintptr_t)b.data - (uintptr_t)a.data);
    if (bytes % size) return true;
    if (ld < std::max(inner_a, inner_b)) return true;
    // b begins q whole lines and r elements past a, 0 <= r < ld: its lines
    // begin on a's q lines on, or (r + inner_b > ld) run into the next ones
    int64_t d = bytes / size, q = d / ld, r = d % ld;
    if (r < 0) r += ld, --q;
    auto lines = [&](int64_t off) { return off < outer_a && -off < outer_b; };
    return (r < inner_a && lines(q)) || (r + inner_b > ld && lines(q + 1));
}

inline bool same(const mxh_mat &a, const mxh_mat &b) {
    return a.data == b.data && (a.rows <= 1 || a.row_stride == b.row_stride) &&
           (a.cols <= 1 || a.col_stride == b.col_stride) && a.rows == b.rows && a.cols == b.cols && a.dtype == b.dtype;
}

inline mxh_mat line(const void *p, int64_t n, int dtype) {
    return mxh_mat{const_cast<void *>(p), 1, n, n, 1, dtype, 0};
}
inline mxh_mat line(const mxh_vec &v) { return line(v.data, v.n, v.dtype); }

inline void refuse_overlap(const mxh_mat &out, const char *a, const mxh_mat &in, const char *b) {
    if (overlap(out, in)) throw Error(std::string(a) + " overlaps " + b);
}

inline void check_workspace(const void *ws, uint64_t have, uint64_t want) {
    if (!want) return;
    if (!ws) throw Error("the call needs " + std::to_string(want) + " bytes of workspace");
    if (have < want)
        throw Error("the call needs " + std::to_string(want) + " bytes of workspace, not " + std::to_string(have));
    if ((uintptr_t)ws % 16) throw Error("workspace: not aligned to 16 bytes");
}

inline void check_act(int act) {
    if (act < MXH_NONE || act > MXH_SIGMOID) throw Error("unknown activation " + std::to_string(act));
}

template <typename F>
int guard(F &&f) {
    try {
        f();
        return 0;
    } catch (const std::exception &e) {
        mx::set_error(e.what());
    } catch (...) {
        mx::set_error("unknown error");
    }
    return -1;
}

// ------------------------------------------------------------- products

// One operand of a product: elements apart along its own axis and along the
// summed one.
struct Operand {
    const void *data;
    int64_t own, sum;
    bool padded;  // lines hold zeros up to whole 16 bytes
    // contiguous along the summed axis ('k') or its own ('m') whatever the
    // strides of axes of one element say; 0: as they say
    char form = 0;
};

// A gated product: the operand along m or n has twice that many lines, the
// gate's and then the values', and results are act(gate) * value.
enum class Pair { kNone, kN, kM };

struct Product {
    int dtype = 0;
    Pair pair = Pair::kNone;
    int64_t m = 0, n = 0, k = 0;
    Operand a{}, b{};
    void *c = nullptr;
    int64_t ldc = 0;
    const mxh_vec *bias = nullptr;
    bool bias_rows = false;
    const void *res = nullptr;
    int64_t ldr = 0;
    void *z = nullptr;
    int64_t ldz = 0;
    const float *back = nullptr;  // fp16: what the sums are multiplied by
    int act = MXH_NONE;
    float slope = 0.0f;
};

struct Plan {
    bool skinny = false;  // the kernel of few rows
    int tile = 0;         // so many lines of both operands
    int bm = 0, bn = 0;  // its results
    unsigned block = 256;
    int stages = 0;  // straight to LDS with so many tiles there; 0: through registers
    bool pack_a = false, pack_b = false;  // copied to aligned lines first
    uint64_t pack_bytes = 0;
    int64_t splits = 1, kchunk = 0;
    uint64_t bytes = 0;
};

// The tile, split and packing of a product, and its workspace.
Plan plan_of(const Product &p);
// Its launches, `ws` of the plan's bytes. `later`: where the sums are cut, not
// the launch that joins them but its arguments (else splits stays 0).
void product(Launches &launches, const Product &p, void *ws, OpsGemmArgs *later = nullptr);
// The launch that joins a plain product's splits.
void join_product(Launches &launches, const OpsGemmArgs &g, int dtype);
// An operand of a product as (own axis, summed axis): rows summed over or not.
Operand operand(const mxh_mat &m, bool sum_rows);

// out[i] = sum over p of part[p][i], two results' sums side by side.
void join(Launches &launches, const float *part, int64_t nparts, int64_t n, void *out0, void *out1, int dtype);

// A product's gradients: the workspace has dz where it is not dy itself, the
// bias's partial sums, and one product's partial sums at a time.
struct BwdLayout {
    mxh_mat dz{};
    int64_t parts = 0;
    uint64_t dz_bytes = 0, part_bytes = 0, top_bytes = 0, product_bytes = 0;
    uint64_t total() const { return dz_bytes + part_bytes + top_bytes + product_bytes; }
};
Product product_dx(const BwdLayout &l, const mxh_mat &w, const mxh_mat &dx);
Product product_dw(const BwdLayout &l, const mxh_mat &x, const mxh_mat &dw);
// dz's blocks along the rows, a partial sum of the bias's gradient each.
int64_t dz_parts(const mxh_mat &dy, bool by_cols);
// dz of dy's positions and so many features, its lines padded to 16 bytes so
// that the products' loads are aligned.
void place_dz(BwdLayout &l, const mxh_mat &dy, int64_t cols, bool by_cols);

inline uint64_t up(uint64_t n) { return (n + 255) / 256 * 256; }

}  // namespace mxops
