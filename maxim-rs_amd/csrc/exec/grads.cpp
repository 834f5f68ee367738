// The gradients' global norm and clipping (include/maxim_block_ops.h): the
// checks of the list, its cut into launches, and the launches.

#include <vector>

#include "../ops/grads_args.h"
#include "maxim_block_ops.h"
#include "ops_host.hpp"

namespace mxops {

// One launch's tensors.
struct GradsLaunch {
    GradsArgs args;
    int64_t grid;
};

static int64_t chunks_of(const mxh_vec &v) { return cdiv(v.n * (int64_t)type_size(v.dtype), MXN_CHUNK); }

static void check_list(const mxh_vec *grads, int64_t count, const char *what) {
    if (count < 0 || count > (1 << 24)) throw Error(std::string(what) + ": " + std::to_string(count) + " tensors");
    if (count && !grads) throw Error(std::string(what) + ": missing");
    for (int64_t i = 0; i < count; ++i) {
        const mxh_vec &v = grads[i];
        const std::string w = std::string(what) + "[" + std::to_string(i) + "]";
        if (v.dtype < MXH_F32 || v.dtype > MXH_BF16) throw Error(w + ": unknown type " + std::to_string(v.dtype));
        if (v.n < 0 || v.n > (int64_t(1) << 44)) throw Error(w + ": " + std::to_string(v.n) + " elements");
        if (v.n && !v.data) throw Error(w + ": no data");
        if ((uintptr_t)v.data % type_size(v.dtype)) throw Error(w + ": not aligned to its element");
    }
}

// The tensors that hold anything, MXN_TENSORS a launch; a launch's chunks have
// 31 bits.
static std::vector<GradsLaunch> cut(const mxh_vec *grads, const mxh_vec *out, int64_t count) {
    std::vector<GradsLaunch> launches;
    int64_t chunks = 0;
    for (int64_t i = 0; i < count; ++i) {
        const int64_t c = chunks_of(grads[i]);
        if (!c) continue;
        if (c >= INT32_MAX) throw Error("grads[" + std::to_string(i) + "]: " + std::to_string(grads[i].n) + " elements");
        if (launches.empty() || launches.back().args.count == MXN_TENSORS || chunks + c >= INT32_MAX) {
            launches.emplace_back();
            launches.back().args.count = 0;
            launches.back().args.first[0] = 0;
            chunks = 0;
        }
        GradsArgs &a = launches.back().args;
        a.src[a.count] = grads[i].data;
        a.dst[a.count] = out ? out[i].data : grads[i].data;
        a.n[a.count] = (uint64_t)grads[i].n | (uint64_t)grads[i].dtype << 56;
        a.first[++a.count] = (uint32_t)(chunks += c);
        // eight blocks of four waves fill a CU
        launches.back().grid = std::min<int64_t>(chunks, 2048);
    }
    return launches;
}

static void launch(int dev, const char *name, int64_t grid, unsigned block, void *stream, void *args) {
    void *params[] = {args};
    check(hip().hipModuleLaunchKernel(function(dev, name), (unsigned)grid, 1, 1, block, 1, 1, 0, (mxh::hipStream_t)stream,
                                      params, nullptr),
          name);
}

static void run_clip(int device, void *stream, std::vector<GradsLaunch> &launches, const float *norm, float max_norm) {
    // last chunks first
    for (size_t i = launches.size(); i-- > 0;) {
        GradsLaunch &l = launches[i];
        l.args.norm = const_cast<float *>(norm);
        l.args.max_norm = max_norm;
        launch(device, "mxn_clip", l.grid, 256, stream, &l.args);
    }
}

// The sum, and clipping, in one launch of one block.
constexpr int64_t kFewChunks = 16;
static bool few(const std::vector<GradsLaunch> &launches) {
    return launches.empty() || (launches.size() == 1 && launches[0].grid <= kFewChunks);
}
static uint64_t norm_bytes(const std::vector<GradsLaunch> &launches) {
    uint64_t n = 0;
    if (!few(launches))
        for (const GradsLaunch &l : launches) n += l.grid * 8;
    return n;
}

// The norm, and where `clip` the results.
static void run(int device, void *stream, std::vector<GradsLaunch> &launches, float *norm, void *workspace, bool clip,
                float max_norm) {
    if (launches.empty()) {  // no elements: the norm alone, 0
        launches.emplace_back();
        launches[0].args.count = 0;
        launches[0].args.first[0] = 0;
    }
    if (few(launches)) {
        GradsArgs &a = launches[0].args;
        a.norm = norm;
        a.clip = clip;
        a.max_norm = max_norm;
        launch(device, "mxn_small", 1, 1024, stream, &a);
        return;
    }
    double *part = static_cast<double *>(workspace);
    for (GradsLaunch &l : launches) {
        l.args.part = part;
        launch(device, "mxn_squares", l.grid, 256, stream, &l.args);
        part += l.grid;
    }
    GradsJoinArgs j{static_cast<double *>(workspace), norm, (int32_t)(part - static_cast<double *>(workspace)), 0};
    launch(device, "mxn_norm", 1, 256, stream, &j);
    if (clip) run_clip(device, stream, launches, norm, max_norm);
}

static void check_norm(const float *norm) {
    if (!norm) throw Error("norm: missing");
    if ((uintptr_t)norm % 4) throw Error("norm: not aligned to its element");
}

// What is written shares no element with anything else of the call, but a
// result with its own gradient, which it replaces.
static void check_apart(const mxh_vec *grads, const mxh_vec *out, int64_t count, const float *norm, bool norm_out) {
    struct Item {
        Range r;
        bool written;
    };
    std::vector<Item> items;
    items.reserve(2 * count + 1);
    auto add = [&](const void *p, uint64_t bytes, bool written) {
        if (bytes) items.push_back({{(uintptr_t)p, (uintptr_t)p + bytes}, written});
    };
    for (int64_t i = 0; i < count; ++i) {
        const uint64_t bytes = (uint64_t)grads[i].n * type_size(grads[i].dtype);
        const bool over = out && out[i].data == grads[i].data;
        if (out) add(out[i].data, bytes, true);
        if (!over) add(grads[i].data, bytes, false);
    }
    add(norm, 4, norm_out);
    std::sort(items.begin(), items.end(), [](const Item &a, const Item &b) { return a.r.lo < b.r.lo; });
    uintptr_t any = 0, written = 0;  // how far those before reach
    for (const Item &i : items) {
        if (i.r.lo < (i.written ? any : written))
            throw Error("a tensor that is written overlaps another one, the norm, or is there twice");
        any = std::max(any, i.r.hi);
        if (i.written) written = std::max(written, i.r.hi);
    }
}

static void check_clip(const mxh_vec *grads, const mxh_vec *&out, int64_t count, float max_norm) {
    check_list(grads, count, "grads");
    if (!(max_norm >= 0.0f)) throw Error("max_norm: not a number of at least 0");
    if (!out) out = grads;
    check_list(out, count, "out");
    for (int64_t i = 0; i < count; ++i)
        if (out[i].n != grads[i].n || out[i].dtype != grads[i].dtype)
            throw Error("out[" + std::to_string(i) + "]: not its gradient's size and type");
}

}  // namespace mxops

using namespace mxops;

extern "C" {

int mxh_grad_norm_workspace(const mxh_vec *grads, int64_t count, uint64_t *bytes) {
    return guard([&] {
        if (!bytes) throw Error("bytes: missing");
        check_list(grads, count, "grads");
        *bytes = norm_bytes(cut(grads, nullptr, count));
    });
}

int mxh_grad_norm(int device, void *stream, const mxh_vec *grads, int64_t count, float *norm, void *workspace,
                  uint64_t workspace_bytes) {
    return guard([&] {
        check_list(grads, count, "grads");
        check_norm(norm);
        check_apart(grads, nullptr, count, norm, true);
        std::vector<GradsLaunch> launches = cut(grads, nullptr, count);
        check_workspace(workspace, workspace_bytes, norm_bytes(launches));
        OnDevice on(device);
        run(device, stream, launches, norm, workspace, false, 0.0f);
    });
}

int mxh_grad_clip(int device, void *stream, const mxh_vec *grads, const mxh_vec *out, int64_t count, float max_norm,
                  float *norm, void *workspace, uint64_t workspace_bytes) {
    return guard([&] {
        check_clip(grads, out, count, max_norm);
        check_norm(norm);
        check_apart(grads, out, count, norm, true);
        std::vector<GradsLaunch> launches = cut(grads, out, count);
        check_workspace(workspace, workspace_bytes, norm_bytes(launches));
        OnDevice on(device);
        run(device, stream, launches, norm, workspace, true, max_norm);
    });
}

int mxh_grad_clip_by(int device, void *stream, const mxh_vec *grads, const mxh_vec *out, int64_t count, float max_norm,
                     const float *norm) {
    return guard([&] {
        check_clip(grads, out, count, max_norm);
        check_norm(norm);
        check_apart(grads, out, count, norm, false);
        std::vector<GradsLaunch> launches = cut(grads, out, count);
        OnDevice on(device);
        run_clip(device, stream, launches, norm, max_norm);
    });
}

}  // extern "C"
