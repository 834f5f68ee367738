// A HIP runtime that runs nothing and writes down the block operators' launches
// (include/maxim_block_ops.h): their host side tested without a device. Built
// twice into one library, with -DDEFAULTS for every entry point's answer of 0
// and without for those below.
#include <cstddef>
#include <cstdint>
#include <cstring>
#include <set>
#include <string>

#include "hip_api.hpp"
#include "../ops/grads_args.h"
#include "../ops/mx4_args.h"

using namespace mxh;

#ifdef DEFAULTS

extern "C" {
#define MXH_FN(ret, name, ...) __attribute__((weak)) ret name(__VA_ARGS__) { return {}; }
#include "hip_api.inc"
}

#else

static std::string g_log;
static std::set<std::string> g_names;
static int g_modules = 0;

static void put(const char *key, long long v) { g_log += std::string(", \"") + key + "\": " + std::to_string(v); }
static void product(const OpsGemmArgs &a) {
    put("a", (intptr_t)a.a), put("b", (intptr_t)a.b), put("lda", a.lda), put("ldb", a.ldb);
    put("m", a.m), put("n", a.n), put("k", a.k), put("splits", a.splits), put("kchunk", a.kchunk);
    put("part", (intptr_t)a.part), put("tiles_m", a.tiles_m), put("tiles_n", a.tiles_n);
}

extern "C" {

hipError_t hipModuleLoadData(hipModule_t *m, const void *) {
    *m = (hipModule_t)(intptr_t)++g_modules;
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
    if ((uint64_t)gx * bx > UINT32_MAX || !gx || !gy) return 9;
    g_log += std::string(g_log.empty() ? "[" : ", ") + "{\"kernel\": \"" + name + "\"";
    put("gx", gx), put("gy", gy), put("block", bx);
    auto begins = [&](const char *p) { return name.rfind(p, 0) == 0; };
    if (begins("mxg_gemm") || begins("mxg_skinny") || begins("mxo_gemm") || begins("mxg_join")) {
        OpsGemmArgs a;
        std::memcpy(&a, params[0], sizeof(a));
        product(a);
    } else if (begins("mxg_dz")) {
        OpsGatedDzArgs g;
        std::memcpy(&g, params[0], sizeof(g));
        const OpsDzArgs &a = g.d;
        put("db", (intptr_t)g.db);
        put("dz", (intptr_t)a.dz), put("part", (intptr_t)a.part), put("nparts", a.nparts), put("drs", a.drs), put("dcs", a.dcs);
    } else if (begins("mxq_gemm") || begins("mxq_skinny")) {
        Mx4GemmArgs a;
        std::memcpy(&a, params[0], sizeof(a));
        product(a.g);
        put("ca", (intptr_t)a.a), put("cb", (intptr_t)a.b), put("sa", (intptr_t)a.sa), put("sb", (intptr_t)a.sb);
    } else if (begins("mxq_")) {
        Mx4CodeArgs a;
        std::memcpy(&a, params[0], sizeof(a));
        put("codes", (intptr_t)a.codes), put("scales", (intptr_t)a.scales), put("tiles", a.tiles);
    } else if (begins("mxn_norm")) {
        GradsJoinArgs a;
        std::memcpy(&a, params[0], sizeof(a));
        put("part", (intptr_t)a.part), put("nparts", a.nparts);
    } else if (begins("mxn_")) {
        GradsArgs a;
        std::memcpy(&a, params[0], sizeof(a));
        put("count", a.count), put("chunks", a.first[a.count]), put("part", (intptr_t)a.part);
        long long n = 0;
        for (int i = 0; i < a.count; ++i) n += a.n[i] & ~(0xffull << 56);
        put("elements", n);
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
int fake_modules(void) { return g_modules; }
}

#endif
