// The training and serving operators' host side (include/maxim_ops.h):
// argument checks, the choice of kernel and split, and the launches. The
// kernels are a code object of their own (csrc/ops), loaded per device by the
// first call.

#include "maxim_ops.h"

#include <algorithm>
#include <array>
#include <cstring>
#include <iterator>
#include <limits>
#include <map>
#include <mutex>
#include <string>
#include <vector>

#include "../ops/ops_args.h"
#include "hip_api.hpp"
#include "host.hpp"

extern "C" const unsigned char mx_ops_hsaco[];

namespace {

using mx::Error;
using mxh::check;
using mxh::hip;

constexpr int kMaxDevices = 64;
constexpr int64_t kMaxExtent = std::numeric_limits<int32_t>::max() - 1024;

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ------------------------------------------------------------ the kernels

struct Code {
    mxh::hipModule_t mod = nullptr;
    std::map<std::string, mxh::hipFunction_t> fns;
};

std::mutex g_mu;
Code g_code[kMaxDevices];

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

mxh::hipFunction_t function(int dev, const std::string &name) {
    auto &H = hip();
    std::lock_guard<std::mutex> lock(g_mu);
    Code &c = g_code[dev];
    if (!c.mod) check(H.hipModuleLoadData(&c.mod, mx_ops_hsaco), "hipModuleLoadData (operators' gfx950 code object)");
    auto it = c.fns.find(name);
    if (it != c.fns.end()) return it->second;
    mxh::hipFunction_t f = nullptr;
    check(H.hipModuleGetFunction(&f, c.mod, name.c_str()), ("hipModuleGetFunction " + name).c_str());
    c.fns[name] = f;
    return f;
}

// A call's launches, of which none is made before all are known to fit: the
// threads of a launch are counted in 32 bits.
class Launches {
    struct One {
        std::string name;
        unsigned gx, gy, block;
        alignas(8) char args[192];
    };
    One at_[8];  // a Dense's backward pass: dz and its join, twice packing, product and join
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
        mxh::hipFunction_t f[8];
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

const char *kTypeName[] = {"f32", "f16", "bf16"};
size_t type_size(int t) { return t == MXH_F32 ? 4 : 2; }

std::string shape(const mxh_mat &m) { return "[" + std::to_string(m.rows) + "][" + std::to_string(m.cols) + "]"; }

bool empty(const mxh_mat &m) { return m.rows == 0 || m.cols == 0; }
// Contiguous along columns (features), or along rows (positions).
bool along_cols(const mxh_mat &m) { return m.col_stride == 1 || m.cols <= 1; }
bool along_rows(const mxh_mat &m) { return m.row_stride == 1 || m.rows <= 1; }

const mxh_mat &need(const mxh_mat *m, const char *what) {
    if (!m) throw Error(std::string(what) + ": missing");
    return *m;
}

void check_mat(const mxh_mat &m, const char *what, int dtype, int64_t rows, int64_t cols) {
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

void check_first(const mxh_mat &x, const char *what) { check_mat(x, what, x.dtype, x.rows, x.cols); }

void check_vec(const mxh_vec &v, const char *what, int64_t n, int dtype) {
    const std::string w = what;
    if (v.n != n) throw Error(w + ": " + std::to_string(v.n) + " elements, expected " + std::to_string(n));
    if (v.dtype != MXH_F32 && v.dtype != dtype) throw Error(w + ": its type is neither fp32 nor x's");
    if (n && !v.data) throw Error(w + ": no data");
    if ((uintptr_t)v.data % type_size(v.dtype)) throw Error(w + ": not aligned to its element");
}

// The memory order that all of a call's matrices have: true, features
// contiguous; false, positions. (One of a single row or column has both.)
bool out_by_cols(const mxh_mat &m) { return along_cols(m) && (m.rows <= 1 || m.row_stride >= m.cols); }
bool out_by_rows(const mxh_mat &m) { return along_rows(m) && (m.cols <= 1 || m.col_stride >= m.rows); }
bool common_order(std::initializer_list<const mxh_mat *> ins, std::initializer_list<const mxh_mat *> outs) {
    bool cols = true, rows = true;
    for (const mxh_mat *m : ins)
        if (m && !empty(*m)) cols = cols && along_cols(*m), rows = rows && along_rows(*m);
    for (const mxh_mat *m : outs)
        if (m && !empty(*m)) cols = cols && out_by_cols(*m), rows = rows && out_by_rows(*m);
    if (!cols && !rows) throw Error("the matrices differ in memory order");
    return cols;
}

// Elements of an output may not share storage.
void check_out(const mxh_mat &m, const char *what) {
    if (empty(m)) return;
    if (!out_by_cols(m) && !out_by_rows(m)) throw Error(std::string(what) + ": elements of an output share storage");
}

struct Range {
    uintptr_t lo, hi;
};
Range range(const mxh_mat &m) {
    const uintptr_t p = (uintptr_t)m.data;
    const uint64_t far = (uint64_t)(m.rows - 1) * m.row_stride + (uint64_t)(m.cols - 1) * m.col_stride + 1;
    return {p, p + far * type_size(m.dtype)};
}
bool apart(Range a, Range b) { return a.hi <= b.lo || b.hi <= a.lo; }

// Whether two views share an element: by their ranges, and where these cross
// and the strides agree (slices of one buffer), by their offset in it.
bool overlap(const mxh_mat &a, const mxh_mat &b) {
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

bool same(const mxh_mat &a, const mxh_mat &b) {
    return a.data == b.data && (a.rows <= 1 || a.row_stride == b.row_stride) &&
           (a.cols <= 1 || a.col_stride == b.col_stride) && a.rows == b.rows && a.cols == b.cols && a.dtype == b.dtype;
}

mxh_mat line(const void *p, int64_t n, int dtype) {
    return mxh_mat{const_cast<void *>(p), 1, n, n, 1, dtype, 0};
}
mxh_mat line(const mxh_vec &v) { return line(v.data, v.n, v.dtype); }

void refuse_overlap(const mxh_mat &out, const char *a, const mxh_mat &in, const char *b) {
    if (overlap(out, in)) throw Error(std::string(a) + " overlaps " + b);
}

void check_workspace(const void *ws, uint64_t have, uint64_t want) {
    if (!want) return;
    if (!ws) throw Error("the call needs " + std::to_string(want) + " bytes of workspace");
    if (have < want)
        throw Error("the call needs " + std::to_string(want) + " bytes of workspace, not " + std::to_string(have));
    if ((uintptr_t)ws % 16) throw Error("workspace: not aligned to 16 bytes");
}

void check_act(int act) {
    if (act < MXH_NONE || act > MXH_SIGMOID) throw Error("unknown activation " + std::to_string(act));
}

// ------------------------------------------------------------- LayerNorm

// The kernel of a LayerNorm pass: by rows, `lpr` threads a row with `nv`
// vectors of 16 bytes each, or in planar order `block` threads, so many lanes
// along the positions and channels a thread; `whole` when the backward kernel
// sums the parameters' gradients too, else another does. `grid` blocks walk
// over the rows; in the backward pass each leaves one partial sum of the
// parameters' gradients.
struct LnPlan {
    std::string form;
    unsigned block = 256;
    int64_t grid = 1;
    bool whole = true;
    int64_t parts = 1;
};

LnPlan ln_plan(int dtype, int64_t rows, int64_t cols, bool by_cols, bool backward) {
    LnPlan p;
    const int64_t e = 16 / (int64_t)type_size(dtype), vecs = cdiv(cols, e);
    if (by_cols) {
        // the fewest threads that hold the row, a vector each: sums stay
        // inside a wave up to 64 vectors
        static const int kForms[][2] = {{8, 1},   {16, 1},  {32, 1},  {64, 1},  {128, 1},
                                        {256, 1}, {512, 1}, {1024, 1}, {1024, 2}};
        for (const auto &f : kForms) {
            if (vecs > f[0] * f[1]) continue;
            p.form = std::to_string(f[0]) + "x" + std::to_string(f[1]);
            p.whole = !(backward && f[1] > 1 && type_size(dtype) == 2);
            p.block = f[0] <= 64 ? 256 : backward ? 1024 : std::max(256, f[0]);
            const int64_t steps = cdiv(rows, p.block / f[0]);
            const int64_t most = 524288 / p.block;
            // a partial sum costs as much as a row: at least eight rows each,
            // once every CU has a block
            p.grid = backward ? std::min(steps, std::max<int64_t>(256, std::min(most / 2, steps / 8))) : std::min(steps, most);
            break;
        }
        if (p.form.empty()) p.form = "long", p.block = 1024, p.grid = std::min<int64_t>(rows, 65536), p.whole = false;
    } else {
        // threads, lanes of 16 bytes along the positions, channels a thread:
        // many lanes where the channels still fit and two tiles a CU are left,
        // else 16 or 8. The backward pass holds two matrices and the
        // parameters' sums: at most eight channels of fp32, four of 16 bits,
        // go into registers. 2^26 bf16 elements: 32 channels with 64 lanes 78
        // us, with 16 177; 64 channels 79 and 94; 128 channels 75 and 66, so
        // 16; 256 channels with 32 lanes 78, with 16 88. Backward, 32 channels
        // with 64 lanes 140 and 16 176; 2^25 floats, 128 channels with 32
        // lanes 95, with 16 88.
        typedef std::vector<std::array<int, 3>> Forms;
        static const Forms kForward16 = {{256, 64, 4}, {256, 64, 8},  {256, 64, 16}, {512, 16, 1},  {512, 16, 2},
                                         {512, 16, 4}, {512, 32, 16}, {512, 16, 8},  {512, 16, 16}, {512, 8, 16}};
        static const Forms kForward32 = {{256, 64, 4}, {256, 64, 8}, {512, 16, 2}, {512, 64, 16}, {512, 32, 16},
                                         {512, 16, 4}, {512, 16, 8}, {512, 16, 16}, {512, 8, 16}};
        static const Forms kBackward16 = {{256, 64, 4}, {512, 64, 4}, {512, 32, 4}, {512, 16, 1},
                                          {512, 16, 2}, {512, 16, 4}, {512, 8, 4}};
        static const Forms kBackward32 = {{256, 64, 4}, {512, 64, 4}, {512, 64, 8}, {512, 16, 1},
                                          {512, 16, 2}, {512, 16, 4}, {512, 16, 8}, {512, 8, 8}};
        int64_t tiles = cdiv(rows, 16 * e);
        for (const auto &f : !backward ? e == 8 ? kForward16 : kForward32 : e == 8 ? kBackward16 : kBackward32) {
            if (cols > f[0] / f[1] * f[2]) continue;
            if (f[1] > 16 && cdiv(rows, f[1] * e) < 512) continue;
            p.form = std::to_string(f[0]) + "x" + std::to_string(f[1]) + "x" + std::to_string(f[2]);
            p.block = f[0];
            tiles = cdiv(rows, f[1] * e);
            p.grid = std::min<int64_t>(tiles, backward ? 262144 / f[0] : 4096);
            break;
        }
        if (p.form.empty()) p.form = "loop", p.block = 512, p.grid = std::min<int64_t>(tiles, 65536), p.whole = false;
    }
    p.grid = std::max<int64_t>(1, p.grid);
    p.parts = p.whole ? p.grid : std::min<int64_t>(256, std::max<int64_t>(1, cdiv(rows, 64)));
    return p;
}

uint64_t ln_bwd_bytes(const mxh_mat &x) {
    if (!x.rows) return 0;
    const int64_t parts = std::max(ln_plan(x.dtype, x.rows, x.cols, true, true).parts,
                                   ln_plan(x.dtype, x.rows, x.cols, false, true).parts);
    return (uint64_t)parts * 2 * x.cols * 4;
}

void join(Launches &launches, const float *part, int64_t nparts, int64_t n, void *out0, void *out1, int dtype) {
    if (!n) return;
    OpsJoinArgs j{};
    j.part = part;
    j.out0 = out0;
    j.out1 = out1;
    j.n = n;
    j.nparts = (int32_t)nparts;
    j.nout = out1 ? 2 : 1;
    j.dtype = dtype;
    launches.add("mxo_join_parts", cdiv(n, 16), j.nout, 1024, j);
}

// ------------------------------------------------------------- products

// One operand of a product: elements apart along its own axis and along the
// summed one.
struct Operand {
    const void *data;
    int64_t own, sum;
    bool padded;  // lines hold zeros up to whole 16 bytes
};

struct Product {
    int dtype = 0;
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
    int act = MXH_NONE;
    float slope = 0.0f;
};

struct Plan {
    bool skinny = false;  // the kernel of few rows
    int bm = 0, bn = 0;
    unsigned block = 256;
    int stages = 0;  // straight to LDS with so many tiles there; 0: through registers
    bool pack_a = false, pack_b = false;  // copied to aligned lines first
    uint64_t pack_bytes = 0;
    int64_t splits = 1, kchunk = 0;
    uint64_t bytes = 0;
};

// How an operand's lines reach the tiles that go straight to LDS: as they lie,
// or copied (`pack` bytes); `ld` elements from line to line there.
struct Side {
    bool by_k;
    uint64_t pack;
    int64_t ld;
};

// Whether a tile of `b` rows (along k) or 128 bytes of k's (along the operand's
// own axis) spans less than 2^31 bytes: its offsets, the size of the buffer
// that bounds it, which has to stay below the offset of lanes without a chunk,
// and the step to the next tile have 31 bits.
bool spans(const Side &s, int64_t b, size_t size) {
    return s.ld < (int64_t(1) << 31) / (s.by_k ? b * (int64_t)size : 128);
}

// What a tile costs, measured in us on square products of 1024 to 8192: a step
// of 128 bytes of k with one tile on a CU (`one`), with as many as its LDS
// holds (`all`, for `fit` of them), and what a tile takes besides.
struct TileCost {
    int b, stages, fit;
    double one, all, rest;
};
const TileCost kTiles16[] = {{256, 2, 1, 1.6, 1.6, 10.0}, {128, 4, 1, 0.54, 0.54, 6.0}, {128, 2, 2, 0.65, 0.93, 7.0},
                             {64, 4, 2, 0.2, 0.39, 4.0},  {128, 0, 2, 1.3, 1.8, 8.0},   {64, 0, 5, 1.1, 1.7, 4.0}};
const TileCost kTiles32[] = {{128, 2, 2, 1.65, 2.95, 8.0}, {64, 4, 2, 0.65, 1.1, 5.0}, {64, 2, 5, 0.75, 2.35, 5.0},
                             {128, 0, 1, 1.95, 1.95, 9.0}, {64, 0, 5, 0.85, 2.6, 6.0}};

// The tile and the number of runs k is cut into that take the least time by
// those costs: rounds of tiles over the 256 CUs, and for a cut k a second
// launch and its partial sums written and read (at 5 TB/s). 4096 x 1024
// results of 4096 products each: 128 x 128 uncut 41 us, cut in two 53 us, 256
// x 256 cut in four 65 us; 1024 x 1024: 64 x 64 uncut 18 us, cut in four 28
// us, 128 x 128 cut in four 26 us.
//
// Up to 16 rows, both operands contiguous along k, can also go to the kernel
// that reads the other operand once, without LDS tiles or a second launch: a
// block for 16 columns and all of k, so it is quick where k is short or there
// are columns enough (0.07 to 0.11 us a step of 128 bytes for every 256 blocks,
// by the rows; the tiles then no faster than the operand comes from memory).
// bf16, one row and 16: k = 4096 to 4096 columns 9.0 and 10.6 us, as tiles 11.6
// and 11.4; k = 1024 to 64 columns 3.8 and 4.5, tiles 5.5 and 5.6; k = 16384 to
// 1024 columns 23 and 31, tiles 12; k = 262144 to 64 columns 334 and 447,
// tiles 14 and 18. fp32, 16 rows: k = 1024 to 4096 columns 7.6, tiles 13; k =
// 4096 to 64 columns 17, tiles 8.4. (The gradient of a planar Dense's weights
// sums over all positions: 32 to 16 features of 448 x 640, fp32, 985 us by few
// rows, 35 by tiles.)
//
// An operand whose tiles cannot go straight to LDS as it lies can be copied to
// aligned lines first (4 us and its bytes twice), which is one more choice:
// 1237 x 1001 x 777 in fp16 takes 22 us through registers. Lines too long for a
// tile's offsets (spans()) go through registers, whose addresses have 64 bits.
Plan plan_product(int dtype, int64_t m, int64_t n, int64_t k, const Side &a, const Side &b) {
    Plan best;
    double least = std::numeric_limits<double>::infinity();
    const int64_t bk = 128 / (int64_t)type_size(dtype), steps = std::max<int64_t>(1, cdiv(k, bk));
    auto consider = [&](const TileCost &t) {
        if (t.stages && !(spans(a, t.b, type_size(dtype)) && spans(b, t.b, type_size(dtype)))) return;
        const uint64_t pack = t.stages ? a.pack + b.pack : 0;
        const int64_t tiles = cdiv(m, t.b) * cdiv(n, t.b);
        for (int64_t cut : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64, 96, 128, 192, 256}) {
            const int64_t each = cdiv(steps, cut), splits = cdiv(steps, each);
            if (cut > 1 && each < 2) continue;
            const int64_t total = tiles * splits, full = total / (256 * t.fit), left = cdiv(total % (256 * t.fit), 256);
            double us = full * (each * t.all + t.rest);
            if (left) us += each * std::max(t.one, t.all * left / t.fit) + t.rest;
            if (splits > 1) us += 5.0 + (double)splits * m * n * 8 / 5e6;
            if (pack) us += 4.0 + 2.0 * pack / 4e6;
            if (us >= least) continue;
            least = us;
            best.bm = best.bn = t.b;
            best.block = t.b == 256 ? 512 : 256;
            best.stages = t.stages;
            best.pack_a = t.stages && a.pack;
            best.pack_b = t.stages && b.pack;
            best.pack_bytes = pack;
            best.splits = splits;
            best.kchunk = each * bk;
        }
    };
    const bool half = type_size(dtype) == 2;
    const TileCost *const tiles = half ? kTiles16 : kTiles32, *const end = half ? std::end(kTiles16) : std::end(kTiles32);
    Plan skinny;
    skinny.skinny = true;
    skinny.block = 512;
    double few = std::numeric_limits<double>::infinity();
    if (a.by_k && b.by_k && m <= 16 && cdiv(n, 16) <= UINT32_MAX / skinny.block) {
        few = 4.0 + (0.065 + 0.0025 * m) * steps * std::max(1.0, cdiv(n, 16) / 256.0);
        // what the tiles take at least, uncut or cut, without trying each cut:
        // a token's call need not wait for that
        double bound = least;
        for (const TileCost *t = tiles; t != end; ++t) bound = std::min(bound, t->rest + std::min(steps * t->one, 2 * t->one + 5.0));
        const double bytes = (double)n * k * type_size(dtype) / 4.9e6;
        if (few <= std::max(bound, bytes)) return skinny;
    }
    for (const TileCost *t = tiles; t != end; ++t) consider(*t);
    if (few <= least) return skinny;
    best.bytes = best.pack_bytes + (best.splits > 1 ? (uint64_t)best.splits * m * n * 4 : 0);
    return best;
}

uint64_t up(uint64_t n) { return (n + 255) / 256 * 256; }

// Contiguous along k (also where there is only one row to stride over), or
// along the operand's own axis.
bool by_k(const Operand &o) { return o.sum == 1; }

// The lines of an operand packed: contiguous extent in whole 16 bytes.
struct Packed {
    int64_t lines, extent, ld;
    uint64_t bytes;
};
Packed packed(bool along_k, int64_t own_n, int64_t sum_n, size_t size) {
    Packed p;
    const int64_t e = 16 / (int64_t)size;
    p.lines = along_k ? own_n : sum_n;
    p.extent = along_k ? sum_n : own_n;
    p.ld = cdiv(p.extent, e) * e;
    p.bytes = up((uint64_t)p.lines * p.ld * size);
    return p;
}

// An operand's tiles go straight to LDS as it lies where 16-byte loads bring
// whole chunks, where lines do not overlap, so that an offset tells what is past
// the end, and where the smallest tile's offsets reach; else from a copy.
Side side(const Operand &o, int64_t own_n, int64_t sum_n, size_t size) {
    const bool k = by_k(o);
    const int64_t e = 16 / (int64_t)size, extent = k ? sum_n : own_n;
    const Side here{k, 0, k ? o.own : o.sum};
    if ((uintptr_t)o.data % 16 == 0 && here.ld % e == 0 && (extent % e == 0 || o.padded) && here.ld >= extent &&
        spans(here, 64, size))
        return here;
    const Packed p = packed(k, own_n, sum_n, size);
    return {k, p.bytes, p.ld};
}

Plan plan_of(const Product &p) {
    if (!p.m || !p.n) return {};
    const size_t size = type_size(p.dtype);
    return plan_product(p.dtype, p.m, p.n, p.k, side(p.a, p.m, p.k, size), side(p.b, p.n, p.k, size));
}

void product(Launches &launches, const Product &given, void *ws) {
    if (!given.m || !given.n) return;
    Product p = given;
    const bool ak = by_k(p.a), bk = by_k(p.b);
    const size_t size = type_size(p.dtype);
    const Plan pl = plan_of(p);
    char *at = static_cast<char *>(ws);
    OpsPackArgs pack{};
    int jobs = 0;
    int64_t blocks = 0;
    auto add = [&](Operand &o, bool along_k, int64_t own_n) {
        const Packed k = packed(along_k, own_n, p.k, size);
        OpsPackJob &j = pack.job[jobs++];
        j.src = o.data;
        j.dst = at;
        j.lines = k.lines, j.extent = k.extent;
        j.src_ld = along_k ? o.own : o.sum;
        j.dst_ld = k.ld;
        const int64_t vecs = k.ld / (16 / (int64_t)size);
        for (j.shift = 3; j.shift < 8 && (int64_t)4 << j.shift < vecs;) ++j.shift;
        j.segs = (int32_t)cdiv(vecs, (int64_t)4 << j.shift);
        blocks = std::max(blocks, cdiv(k.lines, 256 >> j.shift) * j.segs);
        o = along_k ? Operand{at, k.ld, 1, true} : Operand{at, 1, k.ld, true};
        at += k.bytes;
    };
    if (pl.pack_a) add(p.a, ak, p.m);
    if (pl.pack_b) add(p.b, bk, p.n);
    if (jobs) launches.add(size == 2 ? "mxo_pack_16" : "mxo_pack_32", blocks, jobs, 256, pack);
    OpsGemmArgs g{};
    g.a = p.a.data;
    g.b = p.b.data;
    g.c = p.c;
    g.z = p.z;
    g.res = p.res;
    g.part = reinterpret_cast<float *>(at);
    g.lda = ak ? p.a.own : p.a.sum;
    g.ldb = bk ? p.b.own : p.b.sum;
    g.ldc = p.ldc;
    g.ldr = p.ldr;
    g.ldz = p.ldz;
    g.m = (int32_t)p.m;
    g.n = (int32_t)p.n;
    g.k = (int32_t)p.k;
    g.splits = (int32_t)pl.splits;
    g.kchunk = (int32_t)pl.kchunk;
    const std::string t = kTypeName[p.dtype];
    g.act = p.act;
    g.slope = p.slope;
    if (p.bias) {
        g.bias = p.bias->data;
        g.bias_f32 = p.bias->dtype == MXH_F32 && p.dtype != MXH_F32;
        g.bias_rows = p.bias_rows;
    }
    if (pl.skinny) {
        launches.add("mxo_skinny_" + t, cdiv(p.n, 16), 1, pl.block, g);
        return;
    }
    const int64_t tm = cdiv(p.m, pl.bm), tn = cdiv(p.n, pl.bn);
    g.tiles_m = (int32_t)tm;
    g.tiles_n = (int32_t)tn;
    launches.add("mxo_gemm_" + t + "_" + std::to_string(pl.bm) + "x" + std::to_string(pl.bn) + "_" + (ak ? "k" : "m") +
                     (bk ? "k" : "m") + (pl.stages ? "_d" + std::to_string(pl.stages) : ""),
                 tm * tn * pl.splits, 1, pl.block, g);
    if (pl.splits > 1) {
        // few sums of many splits: eight threads to each
        const bool deep = pl.splits >= 16;
        launches.add((deep ? "mxo_join8_" : "mxo_join_") + t,
                     std::min<int64_t>(4096, cdiv(p.m * cdiv(p.n, 4), deep ? 32 : 256)), 1, 256, g);
    }
}

// An operand of a product as (own axis, summed axis): rows summed over or not.
Operand operand(const mxh_mat &m, bool sum_rows) {
    Operand o{m.data, sum_rows ? m.col_stride : m.row_stride, sum_rows ? m.row_stride : m.col_stride, false};
    const int64_t own_n = sum_rows ? m.cols : m.rows, sum_n = sum_rows ? m.rows : m.cols;
    // an axis of one element has no stride of its own: the other one's order
    // holds, and where both are single the element is contiguous
    if (o.sum != 1 && sum_n <= 1 && o.own != 1) o.sum = 1;
    if (o.sum != 1 && o.own != 1 && own_n <= 1) o.own = 1;
    return o;
}

// out = p^T q or p q^T in out's order: rows of `out` run over a's own axis.
Product oriented(const mxh_mat &out, const Operand &rows, const Operand &cols, int64_t k, bool by_cols) {
    Product p;
    p.dtype = out.dtype;
    p.k = k;
    p.c = out.data;
    if (by_cols) {
        p.m = out.rows, p.n = out.cols, p.a = rows, p.b = cols, p.ldc = out.row_stride;
    } else {
        p.m = out.cols, p.n = out.rows, p.a = cols, p.b = rows, p.ldc = out.col_stride;
    }
    return p;
}

Product dense_product(const mxh_mat &x, const mxh_mat &w, const mxh_mat &y, bool by_cols) {
    return oriented(y, operand(x, false), operand(w, false), x.cols, by_cols);
}

// mxh_dense_backward's workspace: dz where there is an activation, the bias's
// partial sums, and one product's partial sums at a time.
struct BwdLayout {
    mxh_mat dz{};
    int64_t parts = 0;
    uint64_t dz_bytes = 0, part_bytes = 0, product_bytes = 0;
    uint64_t total() const { return dz_bytes + part_bytes + product_bytes; }
};

// Blocks enough for the card, 16 rows (or 256 vectors of positions) each at
// least.
int64_t dz_parts(const mxh_mat &dy, bool by_cols) {
    const int64_t e = 16 / (int64_t)type_size(dy.dtype);
    const int64_t across = by_cols ? cdiv(dy.cols, 64 * e) : dy.cols;
    const int64_t most = by_cols ? cdiv(dy.rows, 16) : cdiv(dy.rows, 256 * e);
    return std::max<int64_t>(1, std::min(cdiv(2048, std::max<int64_t>(1, across)), most));
}

// dz as an operand: the pass that writes it fills its lines' ends with zeros.
Operand dz_operand(const BwdLayout &l, bool sum_rows) {
    Operand o = operand(l.dz, sum_rows);
    o.padded = l.dz_bytes != 0;
    return o;
}
Product product_dx(const BwdLayout &l, const mxh_mat &w, const mxh_mat &dx) {
    return oriented(dx, dz_operand(l, false), operand(w, true), w.rows, out_by_cols(dx));
}
Product product_dw(const BwdLayout &l, const mxh_mat &x, const mxh_mat &dw) {
    return oriented(dw, dz_operand(l, true), operand(x, true), x.rows, out_by_cols(dw));
}

BwdLayout bwd_layout(const mxh_mat &dy, bool by_cols, const mxh_mat &x, const mxh_mat &w, const mxh_mat *dx,
                     const mxh_mat *dw, const mxh_vec *db, int act) {
    BwdLayout l;
    l.dz = dy;
    const bool products = dx || dw;
    if (act != MXH_NONE && products) {
        // rows (or planes) padded to 16 bytes, so that the products' loads are
        const int64_t pad = 16 / (int64_t)type_size(dy.dtype);
        if (by_cols) {
            l.dz.row_stride = cdiv(dy.cols, pad) * pad, l.dz.col_stride = 1;
            l.dz_bytes = up((uint64_t)dy.rows * l.dz.row_stride * type_size(dy.dtype));
        } else {
            l.dz.col_stride = cdiv(dy.rows, pad) * pad, l.dz.row_stride = 1;
            l.dz_bytes = up((uint64_t)dy.cols * l.dz.col_stride * type_size(dy.dtype));
        }
        l.dz.data = nullptr;  // aligned wherever the workspace is
    }
    if (db) {
        l.parts = dz_parts(dy, by_cols);
        l.part_bytes = up((uint64_t)l.parts * dy.cols * 4);
    }
    if (dx && !empty(*dx)) l.product_bytes = std::max(l.product_bytes, plan_of(product_dx(l, w, *dx)).bytes);
    if (dw && !empty(*dw)) l.product_bytes = std::max(l.product_bytes, plan_of(product_dw(l, x, *dw)).bytes);
    return l;
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

}  // namespace

extern "C" {

int mxh_ops_ready(int device) {
    return guard([&] {
        OnDevice on(device);
        function(device, "mxo_join_parts");
    });
}

int mxh_layernorm(int device, void *stream, const mxh_mat *x, const mxh_vec *scale, const mxh_vec *bias, float eps,
                  const mxh_mat *y, float *mean, float *rstd) {
    return guard([&] {
        const mxh_mat &X = need(x, "x"), &Y = need(y, "y");
        check_first(X, "x");
        check_mat(Y, "y", X.dtype, X.rows, X.cols);
        check_out(Y, "y");
        if (X.cols == 0) throw Error("x: no columns to normalise over");
        if (!scale) throw Error("scale: missing");
        check_vec(*scale, "scale", X.cols, X.dtype);
        if (bias) {
            check_vec(*bias, "bias", X.cols, X.dtype);
            if (bias->dtype != scale->dtype) throw Error("bias and scale differ in type");
        }
        if (!(eps >= 0.0f)) throw Error("eps: not a number of at least 0");
        const bool by_cols = common_order({x}, {y});
        if (!same(X, Y)) refuse_overlap(Y, "y", X, "x");
        const mxh_mat stats[2] = {line(mean, mean ? X.rows : 0, MXH_F32), line(rstd, rstd ? X.rows : 0, MXH_F32)};
        refuse_overlap(stats[0], "mean", stats[1], "rstd");
        for (const mxh_mat *o : {&Y, &stats[0], &stats[1]}) {
            refuse_overlap(*o, "an output", line(*scale), "scale");
            if (bias) refuse_overlap(*o, "an output", line(*bias), "bias");
            if (o == &Y) continue;
            refuse_overlap(*o, "a statistic", X, "x");
            refuse_overlap(*o, "a statistic", Y, "y");
        }
        if (!X.rows) return;
        OpsLnArgs a{};
        a.x = X.data;
        a.y = Y.data;
        a.scale = scale->data;
        a.bias = bias ? bias->data : nullptr;
        a.mean = mean;
        a.rstd = rstd;
        a.rows = X.rows;
        a.cols = X.cols;
        a.xrs = X.row_stride, a.xcs = X.col_stride;
        a.yrs = Y.row_stride, a.ycs = Y.col_stride;
        a.eps = eps;
        a.param_f32 = scale->dtype == MXH_F32;
        const LnPlan p = ln_plan(X.dtype, X.rows, X.cols, by_cols, false);
        Launches launches;
        launches.add(std::string(by_cols ? "mxo_ln_rows_" : "mxo_ln_planar_") + kTypeName[X.dtype] + "_" + p.form, p.grid,
                     1, p.block, a);
        launches.run(device, stream);
    });
}

int mxh_layernorm_backward_workspace(const mxh_mat *x, uint64_t *bytes) {
    return guard([&] {
        if (!bytes) throw Error("bytes: missing");
        check_first(need(x, "x"), "x");
        *bytes = ln_bwd_bytes(*x);
    });
}

int mxh_layernorm_backward(int device, void *stream, const mxh_mat *dy, const mxh_mat *x, const mxh_vec *scale,
                           const float *mean, const float *rstd, const mxh_mat *add, const mxh_mat *dx,
                           const mxh_vec *dscale, const mxh_vec *dbias, void *workspace, uint64_t workspace_bytes) {
    return guard([&] {
        const mxh_mat &X = need(x, "x"), &DY = need(dy, "dy");
        check_first(X, "x");
        check_mat(DY, "dy", X.dtype, X.rows, X.cols);
        if (X.cols == 0) throw Error("x: no columns to normalise over");
        if (!scale) throw Error("scale: missing");
        check_vec(*scale, "scale", X.cols, X.dtype);
        if (X.rows && (!mean || !rstd)) throw Error("mean, rstd: missing");
        if (add) {
            if (!dx) throw Error("add without dx");
            check_mat(*add, "add", X.dtype, X.rows, X.cols);
        }
        if (dx) {
            check_mat(*dx, "dx", X.dtype, X.rows, X.cols);
            check_out(*dx, "dx");
        }
        if (!dscale != !dbias) throw Error("dscale and dbias come together");
        if (dscale) {
            check_vec(*dscale, "dscale", X.cols, X.dtype);
            check_vec(*dbias, "dbias", X.cols, X.dtype);
            if (dscale->dtype != scale->dtype || dbias->dtype != scale->dtype)
                throw Error("dscale and dbias have scale's type");
        }
        const bool by_cols = common_order({x, dy, add}, {dx});
        const mxh_mat stats[2] = {line(mean, X.rows, MXH_F32), line(rstd, X.rows, MXH_F32)};
        if (dx) {
            if (!same(DY, *dx)) refuse_overlap(*dx, "dx", DY, "dy");
            if (add && !same(*add, *dx)) refuse_overlap(*dx, "dx", *add, "add");
            refuse_overlap(*dx, "dx", X, "x");
            refuse_overlap(*dx, "dx", line(*scale), "scale");
            for (const mxh_mat &s : stats) refuse_overlap(*dx, "dx", s, "the statistics");
        }
        if (dscale) {
            const mxh_mat g[2] = {line(*dscale), line(*dbias)};
            refuse_overlap(g[0], "dscale", g[1], "dbias");
            for (const mxh_mat &o : g) {
                for (const mxh_mat *in : {&X, &DY, dx, add, &stats[0], &stats[1]})
                    if (in) refuse_overlap(o, "a parameter's gradient", *in, "another operand");
                refuse_overlap(o, "a parameter's gradient", line(*scale), "scale");
            }
            check_workspace(workspace, workspace_bytes, ln_bwd_bytes(X));
        }
        Launches launches;
        const std::string t = kTypeName[X.dtype];
        OpsLnBwdArgs a{};
        a.dy = DY.data;
        a.x = X.data;
        a.scale = scale->data;
        a.mean = mean;
        a.rstd = rstd;
        a.part = static_cast<float *>(workspace);
        a.rows = X.rows;
        a.cols = X.cols;
        a.dyrs = DY.row_stride, a.dycs = DY.col_stride;
        a.xrs = X.row_stride, a.xcs = X.col_stride;
        if (add) a.add = add->data, a.ars = add->row_stride, a.acs = add->col_stride;
        if (dx) a.dx = dx->data, a.dxrs = dx->row_stride, a.dxcs = dx->col_stride;
        a.param_f32 = scale->dtype == MXH_F32;
        const LnPlan p = ln_plan(X.dtype, X.rows, X.cols, by_cols, true);
        a.nparts = (int32_t)p.parts;
        const std::string order = by_cols ? "rows_" : "planar_";
        if (X.rows && dscale && !p.whole) {
            // before dx, which may take dy's place
            const int64_t e = by_cols ? 64 * 16 / (int64_t)type_size(X.dtype) : 1;
            launches.add("mxo_ln_param_" + order + t, cdiv(X.cols, e), a.nparts, 256, a);
        }
        if (!dscale) a.part = nullptr;
        if (X.rows && (dx || p.whole)) launches.add("mxo_ln_bwd_" + order + t + "_" + p.form, p.grid, 1, p.block, a);
        if (dscale) join(launches, a.part, X.rows ? p.parts : 0, X.cols, dscale->data, dbias->data, dscale->dtype);
        launches.run(device, stream);
    });
}

int mxh_dense_workspace(const mxh_mat *x, const mxh_mat *w, const mxh_mat *y, uint64_t *bytes) {
    return guard([&] {
        if (!bytes) throw Error("bytes: missing");
        check_first(need(x, "x"), "x");
        check_mat(need(y, "y"), "y", x->dtype, x->rows, need(w, "w").rows);
        // a y of one row or column has both orders, and z or a residual may settle it
        *bytes = 0;
        if (empty(*y)) return;
        if (out_by_cols(*y)) *bytes = plan_of(dense_product(*x, *w, *y, true)).bytes;
        if (out_by_rows(*y)) *bytes = std::max(*bytes, plan_of(dense_product(*x, *w, *y, false)).bytes);
    });
}

int mxh_dense(int device, void *stream, const mxh_mat *x, const mxh_mat *w, const mxh_vec *bias, int act, float slope,
              const mxh_mat *residual, const mxh_mat *y, const mxh_mat *z, void *workspace, uint64_t workspace_bytes) {
    return guard([&] {
        const mxh_mat &X = need(x, "x"), &W = need(w, "w"), &Y = need(y, "y");
        check_first(X, "x");
        check_mat(W, "w", X.dtype, W.rows, X.cols);
        check_mat(Y, "y", X.dtype, X.rows, W.rows);
        check_out(Y, "y");
        check_act(act);
        if (bias) check_vec(*bias, "bias", W.rows, X.dtype);
        if (residual) check_mat(*residual, "residual", X.dtype, X.rows, W.rows);
        if (z) {
            check_mat(*z, "z", X.dtype, X.rows, W.rows);
            check_out(*z, "z");
        }
        const bool by_cols = common_order({residual}, {y, z});
        for (const mxh_mat *o : {y, z}) {
            if (!o) continue;
            refuse_overlap(*o, "an output", X, "x");
            refuse_overlap(*o, "an output", W, "w");
            if (bias) refuse_overlap(*o, "an output", line(*bias), "bias");
            if (residual && !(o == y && same(*residual, Y))) refuse_overlap(*o, "an output", *residual, "the residual");
        }
        if (z) refuse_overlap(Y, "y", *z, "z");
        if (empty(Y)) return;
        Product p = dense_product(X, W, Y, by_cols);
        check_workspace(workspace, workspace_bytes, plan_of(p).bytes);
        p.bias = bias;
        p.bias_rows = !by_cols;
        p.act = act;
        p.slope = slope;
        if (residual) p.res = residual->data, p.ldr = by_cols ? residual->row_stride : residual->col_stride;
        if (z) p.z = z->data, p.ldz = by_cols ? z->row_stride : z->col_stride;
        Launches launches;
        product(launches, p, workspace);
        launches.run(device, stream);
    });
}

int mxh_dense_backward_workspace(const mxh_mat *dy, const mxh_mat *x, const mxh_mat *w, int act, const mxh_mat *dx,
                                 const mxh_mat *dw, const mxh_vec *db, uint64_t *bytes) {
    return guard([&] {
        if (!bytes) throw Error("bytes: missing");
        check_first(need(x, "x"), "x");
        check_mat(need(dy, "dy"), "dy", x->dtype, x->rows, need(w, "w").rows);
        check_act(act);
        *bytes = std::max(bwd_layout(*dy, true, *x, *w, dx, dw, db, act).total(), bwd_layout(*dy, false, *x, *w, dx, dw, db, act).total());
    });
}

int mxh_dense_backward(int device, void *stream, const mxh_mat *dy, const mxh_mat *x, const mxh_mat *w,
                       const mxh_mat *z, int act, float slope, const mxh_mat *dx, const mxh_mat *dw,
                       const mxh_vec *db, void *workspace, uint64_t workspace_bytes) {
    return guard([&] {
        const mxh_mat &X = need(x, "x"), &W = need(w, "w"), &DY = need(dy, "dy");
        check_first(X, "x");
        check_mat(W, "w", X.dtype, W.rows, X.cols);
        check_mat(DY, "dy", X.dtype, X.rows, W.rows);
        check_act(act);
        if (act != MXH_NONE && !z) throw Error("z: missing (the activation's derivative needs it)");
        if (act == MXH_NONE) z = nullptr;
        if (z) check_mat(*z, "z", X.dtype, X.rows, W.rows);
        if (dx) {
            check_mat(*dx, "dx", X.dtype, X.rows, X.cols);
            check_out(*dx, "dx");
        }
        if (dw) {
            check_mat(*dw, "dw", X.dtype, W.rows, W.cols);
            check_out(*dw, "dw");
        }
        if (db) check_vec(*db, "db", W.rows, X.dtype);
        // z may settle the order of a dy of one row or column
        const bool dz_cols = common_order({dy, z}, {});
        const mxh_mat dbl = db ? line(*db) : mxh_mat{};
        const mxh_mat *outs[] = {dx, dw, db ? &dbl : nullptr}, *ins[] = {dy, x, w, z};
        const char *on_[] = {"dx", "dw", "db"}, *in_[] = {"dy", "x", "w", "z"};
        for (int i = 0; i < 3; ++i) {
            if (!outs[i]) continue;
            for (int j = 0; j < 4; ++j)
                if (ins[j]) refuse_overlap(*outs[i], on_[i], *ins[j], in_[j]);
            for (int j = 0; j < i; ++j)
                if (outs[j]) refuse_overlap(*outs[i], on_[i], *outs[j], on_[j]);
        }
        BwdLayout l = bwd_layout(DY, dz_cols, X, W, dx, dw, db, act);
        check_workspace(workspace, workspace_bytes, l.total());
        Launches launches;
        char *ws = static_cast<char *>(workspace);
        const std::string t = kTypeName[X.dtype];
        OpsDzArgs a{};
        a.dy = DY.data;
        a.rows = DY.rows;
        a.cols = DY.cols;
        a.dyrs = DY.row_stride, a.dycs = DY.col_stride;
        if (z) a.z = z->data, a.zrs = z->row_stride, a.zcs = z->col_stride;
        if (l.dz_bytes) l.dz.data = a.dz = ws, a.drs = l.dz.row_stride, a.dcs = l.dz.col_stride;
        if (db) a.part = reinterpret_cast<float *>(ws + l.dz_bytes);
        a.nparts = (int32_t)dz_parts(DY, dz_cols);
        a.act = act;
        a.slope = slope;
        if ((a.dz || a.part) && !empty(DY))
            launches.add((dz_cols ? "mxo_dz_rows_" : "mxo_dz_planar_") + t,
                         dz_cols ? cdiv(DY.cols, 64 * 16 / (int64_t)type_size(DY.dtype)) : DY.cols, a.nparts, 256, a);
        if (db) join(launches, a.part, DY.rows ? l.parts : 0, DY.cols, db->data, nullptr, db->dtype);
        void *pw = ws + l.dz_bytes + l.part_bytes;
        if (dx && !empty(*dx)) product(launches, product_dx(l, W, *dx), pw);
        if (dw && !empty(*dw)) product(launches, product_dw(l, X, *dw), pw);
        launches.run(device, stream);
    });
}

}  // extern "C"
