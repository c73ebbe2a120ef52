// Stand-in for the runner's side of the seam of sgemm_i8.cpp: records launches and tensor maps instead of making them.
#include "sgemm_internal.hpp"

#include <cstring>
#include <string>

struct sgemm_handle {
    bool int8 = false;
    int64_t force = 0, split = 0;
};

namespace {
struct Launch {
    uint32_t count;
    int32_t function;
    uint32_t grid, threads, smem, cluster, maps, box[4];
    uint64_t dims[4];
    int32_t variant;
    uint32_t parts, tile_n, tpr;
};
sgemm_handle g_handle;
Launch g_last;
std::string g_error;
uint32_t g_maps = 0;
int g_scopes = 0;   // contexts made current and not put back
void *g_functions[sgemm_internal::kI8Functions];
uint32_t g_status[16];
}  // namespace

namespace sgemm_internal {

int set_error(sgemm_handle *, int code, const char *message) {
    g_error = message;
    return code;
}
bool i8_view(sgemm_handle *h, I8View *v) {
    if (!h->int8) return false;
    for (int i = 0; i < kI8Functions; ++i) g_functions[i] = reinterpret_cast<void *>((uintptr_t)i + 1);
    v->functions = g_functions;
    v->status = g_status;
    v->sm_count = 148;
    v->tile_n = 256;
    v->main_smem = 6 * 32768 + 1280;
    v->force_variant = h->force;
    v->split_k = h->split;
    const uint32_t fit[5] = {0, 74, 33, 22, 15};   // what a B200 holds
    for (int i = 0; i < 5; ++i) v->wgrad_clusters[i] = fit[i];
    return true;
}
I8Scope::I8Scope(sgemm_handle *) : pushed_(true) { ++g_scopes; }
I8Scope::~I8Scope() { g_scopes -= pushed_; }

int i8_launch(sgemm_handle *, void *function, uint32_t grid, uint32_t threads, uint32_t smem, uint32_t cluster, void *, void **params) {
    if (g_scopes != 1) return -4;   // as the driver: no current context
    ++g_last.count;
    g_last.function = (int32_t)(reinterpret_cast<uintptr_t>(function) - 1);
    g_last.grid = grid;
    g_last.threads = threads;
    g_last.smem = smem;
    g_last.cluster = cluster;
    g_last.maps = g_maps;
    g_maps = 0;
    if (std::strncmp(i8_function_name(g_last.function), "i8_quantize", 11) == 0 || std::strncmp(i8_function_name(g_last.function), "i8_rmsnorm", 10) == 0) {
        // six pointers, then k, rows, ldx, ldr, lds, ldq, tpr
        g_last.tpr = reinterpret_cast<const uint32_t *>(static_cast<const char *>(params[0]) + 6 * sizeof(void *))[6];
    }
    return 0;
}
int i8_encode(sgemm_handle *, I8TensorMap *, I8MapType, const void *, uint64_t d0, uint64_t d1, uint64_t, uint32_t b0, uint32_t b1, bool) {
    if (g_scopes != 1) return -4;
    if (g_maps < 2) {
        g_last.dims[2 * g_maps] = d0;
        g_last.dims[2 * g_maps + 1] = d1;
        g_last.box[2 * g_maps] = b0;
        g_last.box[2 * g_maps + 1] = b1;
    }
    ++g_maps;
    return 0;
}
void i8_note(sgemm_handle *, int variant, uint32_t parts, uint32_t, uint32_t tile_n) {
    g_last.variant = variant;
    g_last.parts = parts;
    g_last.tile_n = tile_n;
}

}  // namespace sgemm_internal

extern "C" {
void *seam_handle(int int8, int64_t force, int64_t split) {
    g_handle = sgemm_handle{int8 != 0, force, split};
    g_last = Launch{};
    g_maps = 0;
    return &g_handle;
}
void seam_last(Launch *out) { *out = g_last; }
const char *seam_error() { return g_error.c_str(); }
const char *seam_name(int index) { return sgemm_internal::i8_function_name(index); }
int seam_count() { return sgemm_internal::i8_function_count(); }
int seam_registers(int index) { return sgemm_internal::i8_function_registers(index); }
}
