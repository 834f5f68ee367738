// A HIP runtime that runs nothing and writes down what it is asked to launch:
// the operators' host side (csrc/exec/ops.cpp) tested without a device. Built
// twice into one library, with -DDEFAULTS for every entry point's answer of 0
// and without for those below.
#include <cstdint>
#include <cstddef>
#include <cstdio>
#include <cstring>
#include <set>
#include <string>

#include "hip_api.hpp"
#include "../ops/ops_args.h"

using namespace mxh;

#ifdef DEFAULTS

extern "C" {
#define MXH_FN(ret, name, ...) __attribute__((weak)) ret name(__VA_ARGS__) { return {}; }
#include "hip_api.inc"
}

#else

static std::string g_log;
static std::set<std::string> g_names;

static void put(const char *key, long long v) { g_log += std::string(", \"") + key + "\": " + std::to_string(v); }

extern "C" {

hipError_t hipModuleLoadData(hipModule_t *m, const void *) {
    *m = (hipModule_t)1;
    return 0;
}
hipError_t hipModuleGetFunction(hipFunction_t *f, hipModule_t, const char *name) {
    *f = (hipFunction_t)g_names.insert(name).first->c_str();
    return 0;
}
const char *hipGetErrorString(hipError_t) { return "refused by the fake runtime"; }

hipError_t hipModuleLaunchKernel(hipFunction_t f, unsigned gx, unsigned gy, unsigned, unsigned bx, unsigned, unsigned,
                                 unsigned, hipStream_t, void **params, void **) {
    const std::string name = (const char *)f;
    // as the real one: the threads along x have to fit 32 bits
    if ((uint64_t)gx * bx > UINT32_MAX) return 9;
    g_log += std::string(g_log.empty() ? "[" : ", ") + "{\"kernel\": \"" + name + "\"";
    put("gx", gx), put("gy", gy), put("block", bx);
    if (name.rfind("mxo_gemm", 0) == 0 || name.rfind("mxo_skinny", 0) == 0) {
        OpsGemmArgs a;
        std::memcpy(&a, params[0], sizeof(a));
        put("a", (intptr_t)a.a), put("b", (intptr_t)a.b), put("lda", a.lda), put("ldb", a.ldb);
        put("m", a.m), put("n", a.n), put("k", a.k), put("splits", a.splits), put("kchunk", a.kchunk);
        put("part", (intptr_t)a.part);
    } else if (name.rfind("mxo_pack", 0) == 0) {
        OpsPackArgs a;
        std::memcpy(&a, params[0], sizeof(a));
        for (unsigned i = 0; i < gy; ++i) {
            const std::string n = std::to_string(i);
            put(("dst" + n).c_str(), (intptr_t)a.job[i].dst);
            put(("end" + n).c_str(), (intptr_t)a.job[i].dst + a.job[i].lines * a.job[i].dst_ld * (name.back() == '6' ? 2 : 4));
        }
    }
    g_log += "}";
    return 0;
}

// The launches since the last call, as JSON.
const char *fake_launches(void) {
    static std::string out;
    out = g_log.empty() ? "[]" : g_log + "]";
    g_log.clear();
    return out.c_str();
}
}

#endif
