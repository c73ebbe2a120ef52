// The 8-bit entry points of libsgemm_runner.so (include/sgemm_runner.h, "8-bit operands"): argument checks, the choice
// of kernel and cut, tensor maps and launches.  They work on handles of cubins generated for INT8 operands.
//
// Every call is one launch.  None of them uses the handle's workspace or keeps anything between calls: tensor maps are made
// anew from the arguments and travel as kernel arguments, parts of a cut sum meet in shared memory.  So calls on several
// streams, and captured graphs replayed side by side, need no ordering among themselves beyond that of their data.
#include "sgemm_internal.hpp"
#include "sgemm_i8_params.hpp"

#include <algorithm>
#include <cstdio>
#include <cstring>
#include <utility>

#define SGEMM_API extern "C" __attribute__((visibility("default")))

namespace {

using namespace sgemm_internal;

constexpr uint32_t kSmsPerPair = 2;

// index of a kernel in the handle's table; the row kernels follow as [operation][type][form]
enum : int {
    kFew16 = 0, kFew32, kFew64, kFew128, kWgrad, kWgradSimt, kLinear, kHalf, kLinearSimt,
    kQuantize,                                   // + 5 * type + form (8, 16, 32 elements per thread in aligned vectors; shifted vectors; single elements)
    kNorm = kQuantize + 15,
    kRestore = kNorm + 15,                       // + 2 * type + (0 aligned vectors, 1 shifted ones)
    kCount = kRestore + 6
};
static_assert(kCount <= kI8Functions, "the handle's table holds every kernel");

const char *const kNames[kCount] = {
    "i8_linear_few_16", "i8_linear_few_32", "i8_linear_few_64", "i8_linear_few_128", "i8_wgrad", "i8_wgrad_simt",
    "generated_gemm", "i8_linear_half", "generated_gemm_simt",
    "i8_quantize_fp32_v1", "i8_quantize_fp32_v2", "i8_quantize_fp32_v4", "i8_quantize_fp32_u4", "i8_quantize_fp32_s4",
    "i8_quantize_fp16_v1", "i8_quantize_fp16_v2", "i8_quantize_fp16_v4", "i8_quantize_fp16_u4", "i8_quantize_fp16_s4",
    "i8_quantize_bf16_v1", "i8_quantize_bf16_v2", "i8_quantize_bf16_v4", "i8_quantize_bf16_u4", "i8_quantize_bf16_s4",
    "i8_rmsnorm_fp32_v1", "i8_rmsnorm_fp32_v2", "i8_rmsnorm_fp32_v4", "i8_rmsnorm_fp32_u4", "i8_rmsnorm_fp32_s4",
    "i8_rmsnorm_fp16_v1", "i8_rmsnorm_fp16_v2", "i8_rmsnorm_fp16_v4", "i8_rmsnorm_fp16_u4", "i8_rmsnorm_fp16_s4",
    "i8_rmsnorm_bf16_v1", "i8_rmsnorm_bf16_v2", "i8_rmsnorm_bf16_v4", "i8_rmsnorm_bf16_u4", "i8_rmsnorm_bf16_s4",
    "i8_restore_fp32_v", "i8_restore_fp32_u", "i8_restore_fp16_v", "i8_restore_fp16_u", "i8_restore_bf16_v", "i8_restore_bf16_u",
};

struct FewKernel {
    int index;
    uint32_t tile_n, smem;
};
const FewKernel kFew[] = {
    {kFew16, 16, I8_FEW_SMEM(16, I8_FEW_STAGES_16)},
    {kFew32, 32, I8_FEW_SMEM(32, I8_FEW_STAGES_32)},
    {kFew64, 64, I8_FEW_SMEM(64, I8_FEW_STAGES_64)},
    {kFew128, 128, I8_FEW_SMEM(128, I8_FEW_STAGES_128)},
};

// mirrors of the kernels' argument structures
struct LinearArgs {
    const void *w, *sw, *x, *sx, *bias;
    void *y;
    uint32_t *status;
    uint32_t m, n, k, ldw, ldx, ldy, y_type, tiles_m, tiles_n;
};
struct WgradArgs {
    const void *q, *scale, *g, *c;
    void *d;
    uint32_t *status;
    uint32_t m, n, tokens, ldq, ldg, ldc, ldd, g_type, d_type;
    float alpha, beta;
    uint32_t tiles_m, tiles_n;
};
struct RowArgs {
    const void *x, *r, *g;
    void *sum, *q, *scale;
    uint32_t k, rows, ldx, ldr, lds, ldq, tpr, tpr_log2, passes, pow2;
    float eps, inv_k;
};

int refuse(sgemm_handle *h, int code, const char *op, const char *what) {
    char text[256];
    std::snprintf(text, sizeof text, "%s: %s", op, what);
    return set_error(h, code, text);
}
uint32_t ceil_div(uint32_t a, uint32_t b) { return (a + b - 1) / b; }   // (a + b - 1 stays below 2^32: callers bound a)
bool aligned(const void *p, size_t bytes) { return ((uintptr_t)p % bytes) == 0; }
uint32_t type_bytes(int type) { return type == (int)SGEMM_I8_FP32 ? 4u : 2u; }
bool known_type(int type) { return type >= 0 && type <= 2; }

// what every entry point checks first
int begin(sgemm_handle *h, const char *op, I8View *v) {
    if (!h) return SGEMM_ERR_INVALID_ARGUMENT;
    if (!i8_view(h, v)) return refuse(h, SGEMM_ERR_UNSUPPORTED, op, "the loaded cubin is not one for INT8 operands");
    return SGEMM_OK;
}

constexpr uint32_t kLargest = 0x7FFFFF00u;   // sizes above this would leave 31 bits when rounded up to a tile

constexpr uint32_t kLongestRow = 1u << 30;   // the row kernels count a row's elements in 32 bits with a sign

// ---------------------------------------------------------------------------------------------- linear
struct LinearPlan {
    int index = kLinear;
    const FewKernel *few = nullptr;
    uint32_t parts = 1;
};

// Estimated nanoseconds of a call on each kernel, fitted to calls back to back on a B200 (captured graphs, weights out of L2).  What matters
// is where they cross: (tokens, channels, features) = (509, 4096, 4096) takes 14.9 us on 256 x 256 tiles, 10.8 on 256 x 128
// and 14.2 on 128 x 128; (1024, 4096, 4096) 15.8, 17.2 and 26.8; (64, 4096, 4096) 14.8, 10.0 and, cut in 4 parts, 9.2.  Over 112 shapes of 4096 to
// 151936 channels, 2048 to 28672 features and 1 to 128 tokens the kernel of the least estimate is within 10 % of the fastest of all, 0.4 % on
// average.  (Over 320 random ones, whose features end inside a 128-byte line, its time is up to 23 % above that of the pairs: the
// estimates know nothing of the lines.)
//   pairs: set-up and the first loads, then so many waves of tiles with a stage every 320 ns (256 x 256) or 190 (256 x 128)
uint64_t pair_ns(uint64_t tiles, uint32_t pairs, uint32_t stages, bool half) {
    const uint64_t waves = (tiles + pairs - 1) / pairs;
    return half ? 4400 + waves * stages * 190 : 5000 + waves * stages * 320;
}
//   ... and never below the trip of its `bytes` from memory, which with the few large tiles of wide outputs is a little slower than with the
//   few-token kernels' many: 256 x 128 tiles against 128 x 16 take 47.6 us and 41.5 for (1, 28672, 8192), 15.1 and 11.7 for (1, 12288, 4096);
//   against 128 x 64 tiles 45.7 and 44.6 for (64, 28672, 8192), 13.1 and 13.9 for (64, 12288, 4096)
uint64_t pair_trip_ns(uint64_t bytes) { return 4500 + bytes / 6000; }
//   few tokens: a stage's cost is the latency of its loads over the depth of the ring; a cut adds the cluster's barriers and the sum over
//   the parts, and is limited by how many clusters the device holds (148 SMs in uneven groups): a second wave of clusters begins when the first
//   has added up, (1, 28672, 4096) takes 22.2 us whole, 25.8 in 2 parts, 40.3 in 8.  Never below the trip from memory; where that decides, the
//   cut with more loads under way is a little faster
uint64_t few_ns(const FewKernel &f, uint64_t tiles, uint32_t stages, uint32_t parts, uint32_t sms, uint64_t bytes) {
    const uint32_t per_sm = f.tile_n <= 64 ? 2 : 1;
    const uint64_t slots = std::max<uint64_t>(per_sm * (parts == 1 ? sms : parts == 2 ? sms / 2 : parts == 4 ? sms * 33 / 148 : sms * 15 / 148), 1);
    const uint64_t waves = (tiles + slots - 1) / slots;
    const uint64_t stage = f.tile_n == 128 ? 345 : f.tile_n == 64 ? 317 : f.tile_n == 32 ? 270 : 236;
    const uint64_t ns = 2000 + waves * ceil_div(stages, parts) * stage + (parts > 1 ? 1100 + 40ull * f.tile_n : 0);
    const uint64_t trip = 3500 + bytes / 6600 + (parts > 1 ? 30 : 10) * f.tile_n;
    return std::max(ns, trip) + ns / 8 + (waves - 1) * (parts == 1 ? 20 * f.tile_n : trip > ns ? 2000 : 0);
}

int plan_linear(sgemm_handle *h, const I8View &v, const void *w, const void *x, uint32_t m, uint32_t n, uint32_t k,
                uint32_t ldw, uint32_t ldx, int y_type, LinearPlan *p) {
    const bool tma = aligned(w, 16) && aligned(x, 16) && ldw % 16 == 0 && ldx % 16 == 0;
    if (v.force_variant != 0 && v.force_variant != 2 && (!tma || k == 0))
        return refuse(h, SGEMM_ERR_UNSUPPORTED, "sgemm_i8_linear",
                      "a tensor kernel is forced but the operands need 16-byte aligned bases, leading dimensions that are multiples of 16 and K > 0");
    if (v.force_variant == 2 || !tma || k == 0) {
        p->index = kLinearSimt;
        return SGEMM_OK;
    }
    p->index = v.force_variant == 4 ? kHalf : kLinear;
    if (v.force_variant == 1 || v.force_variant == 4) return SGEMM_OK;
    const uint32_t sms = (uint32_t)std::max(v.sm_count, 2), pairs = sms / kSmsPerPair, stages = ceil_div(k, I8_BK);
    const uint64_t full = pair_ns((uint64_t)ceil_div(m, 256) * ceil_div(n, v.tile_n), pairs, stages, false);
    const uint64_t half = pair_ns((uint64_t)ceil_div(m, 256) * ceil_div(n, I8_HALF_BN), pairs, stages, true);
    const uint64_t bytes = (uint64_t)m * k + (uint64_t)n * k + (uint64_t)m * n * type_bytes(y_type);
    uint64_t best = std::max(std::min(full, half), pair_trip_ns(bytes));
    if (half < full) p->index = kHalf;
    // the few-token kernel whose tile holds all tokens (the widest takes more than one tile only when it is forced)
    const FewKernel *few = &kFew[3];
    for (const FewKernel &f : kFew)
        if (n <= f.tile_n) { few = &f; break; }
    const uint64_t tiles = (uint64_t)ceil_div(m, I8_BM) * ceil_div(n, few->tile_n);
    if (v.force_variant == 3) best = ~0ull;
    else if (n > few->tile_n) return SGEMM_OK;
    for (uint32_t parts = 1; parts <= 8; parts *= 2) {
        if (v.split_k > 0 && parts != (v.split_k >= 8 ? 8u : v.split_k >= 4 ? 4u : v.split_k >= 2 ? 2u : 1u)) continue;
        if (v.split_k == 0 && parts > 1 && stages < 2 * parts) break;
        const uint64_t ns = few_ns(*few, tiles, stages, parts, sms, bytes);
        if (ns < best) {
            best = ns;
            p->index = few->index;
            p->few = few;
            p->parts = parts;
        }
    }
    return SGEMM_OK;
}

// ------------------------------------------------------------------------------------------ row kernels
// How the rows lie: all in aligned vectors; all starting at the same offset into one (so that one thread's elements are one vector of
// each); or anyhow.
enum RowForm { kRowsAligned, kRowsShifted, kRowsAnyhow };

// Threads per row and elements per thread.  With many rows 32 elements a thread (256 threads hold 8192; longer rows are read twice);
// while all rows together leave SMs short of threads, twice the threads with half the elements, down to 8: a few rows are
// a matter of latency.
void plan_rows(const I8View &v, uint32_t k, uint32_t rows, RowForm form, uint32_t *tpr, int *kernel) {
    uint32_t per = 32, threads = 32;
    const uint32_t elements = form == kRowsShifted ? k + 7 : k;   // (a shifted row reaches into one vector more)
    while (threads < 256 && threads * per < elements) threads *= 2;
    if (form == kRowsAligned) {
        while (per > 8 && threads * per >= k / 2 && (uint64_t)rows * threads < (uint64_t)v.sm_count * 1024) {
            threads *= 2;
            per /= 2;
        }
        while (per > 8 && threads * (per / 2) >= k) per /= 2;
    }
    *tpr = threads;
    *kernel = form == kRowsAnyhow ? 4 : form == kRowsShifted ? 3 : per == 32 ? 2 : per == 16 ? 1 : 0;
}

// rows of `type` and their int8 images: x and, where there are, the residual and the sum
RowForm row_form(int type, const RowArgs &a) {
    const uint32_t eb = type_bytes(type), per = 16 / eb;
    bool is_aligned = aligned(a.q, per) && a.ldq % per == 0 && (!a.g || aligned(a.g, 16)), alike = true;
    const std::pair<const void *, uint32_t> rows[3] = {{a.x, a.ldx}, {a.r, a.ldr}, {a.sum, a.lds}};
    for (const auto &m : rows) {
        if (!m.first) continue;
        is_aligned = is_aligned && aligned(m.first, 16) && (uint64_t)m.second * eb % 16 == 0;
        alike = alike && ((uintptr_t)m.first - (uintptr_t)a.x) % 16 == 0 && ((uint64_t)m.second - a.ldx) * eb % 16 == 0;
    }
    return is_aligned ? kRowsAligned : alike ? kRowsShifted : kRowsAnyhow;
}

int launch_rows(sgemm_handle *h, const I8View &v, int base, int type, RowArgs &a, void *stream) {
    I8Scope scope(h);
    int kernel = 0;
    const RowForm form = row_form(type, a);
    plan_rows(v, a.k, a.rows, form, &a.tpr, &kernel);
    const uint32_t span = a.tpr * (kernel == 0 ? 8 : kernel == 1 ? 16 : 32);
    const uint32_t reach = a.k + (form == kRowsShifted ? 16 / type_bytes(type) - 1 : 0);   // of a shifted row from its first vector on
    a.passes = std::max(1u, ceil_div(reach, span));
    for (a.tpr_log2 = 0; (1u << a.tpr_log2) < a.tpr;) ++a.tpr_log2;
    a.inv_k = a.k ? 1.0f / (float)a.k : 0.0f;
    const uint32_t threads = std::max<uint32_t>(I8_ROW_THREADS, a.tpr), per_block = threads / a.tpr;
    void *params[] = {&a};
    return i8_launch(h, v.functions[base + 5 * type + kernel], ceil_div(a.rows, per_block), threads, 0, 0, stream, params);
}

}  // namespace

namespace sgemm_internal {

int i8_function_count() { return kCount; }
const char *i8_function_name(int index) { return kNames[index]; }
uint32_t i8_function_smem(int index, uint32_t main_smem) {
    for (const FewKernel &f : kFew)
        if (f.index == index) return f.smem;
    return index == kWgrad ? (uint32_t)I8W_SMEM : index == kLinear ? main_smem : index == kHalf ? (uint32_t)I8_PAIR_SMEM(I8_HALF_BN, I8_HALF_STAGES) : 0u;
}
int i8_wgrad_function() { return kWgrad; }
uint32_t i8_wgrad_threads() { return I8W_THREADS; }
const uint32_t *i8_layout(size_t *words) {
    static const uint32_t layout[SGEMM_I8_LAYOUT_WORDS] = SGEMM_I8_LAYOUT;
    *words = SGEMM_I8_LAYOUT_WORDS;
    return layout;
}
int i8_function_registers(int index) { return index == kWgrad ? I8W_LAUNCH_REGS : 0; }

}  // namespace sgemm_internal

SGEMM_API int sgemm_i8_linear(sgemm_handle *h, const int8_t *dW, const float *dWscale, const int8_t *dX, const float *dXscale,
                              const float *dBias, void *dY, int y_type, uint32_t m, uint32_t n, uint32_t k, uint32_t ldw,
                              uint32_t ldx, uint32_t ldy, void *stream) {
    const char *op = "sgemm_i8_linear";
    I8View v;
    int rc = begin(h, op, &v);
    if (rc) return rc;
    if (!known_type(y_type)) return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "Y's type is FP32 (0), FP16 (1) or BF16 (2)");
    if (k > I8_MAX_K) return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "K above 131071: the 32-bit integer sum could overflow");
    if (ldw < std::max(k, 1u) || ldx < std::max(k, 1u) || ldy < std::max(m, 1u))
        return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "a leading dimension is smaller than the rows it must hold");
    if (m == 0 || n == 0) return SGEMM_OK;
    if (m > kLargest || n > kLargest) return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "problem too large");
    if (!dWscale || !dXscale || !dY || (k && (!dW || !dX))) return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "a matrix or its scales are NULL");
    if (!aligned(dY, type_bytes(y_type))) return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "Y is not aligned to its element type");
    if (!aligned(dWscale, 4) || !aligned(dXscale, 4) || !aligned(dBias, 4))
        return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "scales and bias are FP32 and must be aligned to 4 bytes");
    I8Scope scope(h);
    LinearPlan p;
    if ((rc = plan_linear(h, v, dW, dX, m, n, k, ldw, ldx, y_type, &p))) return rc;
    LinearArgs a{dW, dWscale, dX, dXscale, dBias, dY, v.status, m, n, k, ldw, ldx, ldy, (uint32_t)y_type, 0, 0};
    const bool pair = p.index == kLinear || p.index == kHalf;
    const uint32_t tile_m = pair ? 256 : p.few ? I8_BM : I8_SIMT_TILE;
    const uint32_t tile_n = p.index == kLinear ? v.tile_n : p.index == kHalf ? I8_HALF_BN : p.few ? p.few->tile_n : I8_SIMT_TILE;
    a.tiles_m = ceil_div(m, tile_m);
    a.tiles_n = ceil_div(n, tile_n);
    const uint64_t tiles = (uint64_t)a.tiles_m * a.tiles_n;
    if (tiles * p.parts > 0x7FFFFFFFull) return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "problem too large");
    if (p.index == kLinearSimt) {
        void *params[] = {&a};
        rc = i8_launch(h, v.functions[kLinearSimt], (uint32_t)tiles, I8_SIMT_THREADS, 0, 0, stream, params);
        i8_note(h, 2, 1, (uint32_t)tiles, tile_n);
        return rc;
    }
    I8TensorMap map_w, map_x;
    const uint32_t box_n = p.few ? tile_n : tile_n / 2;
    if ((rc = i8_encode(h, &map_w, kMapInt8, dW, k, m, ldw, I8_BK, I8_BM, true))) return rc;
    if ((rc = i8_encode(h, &map_x, kMapInt8, dX, k, n, ldx, I8_BK, box_n, true))) return rc;
    void *params[] = {&a, &map_w, &map_x};
    if (p.few) {
        rc = i8_launch(h, v.functions[p.index], (uint32_t)tiles * p.parts, I8_FEW_THREADS, p.few->smem, p.parts, stream, params);
        i8_note(h, 3, p.parts, (uint32_t)tiles * p.parts, tile_n);
        return rc;
    }
    const uint32_t grid = kSmsPerPair * (uint32_t)std::min<uint64_t>(tiles, (uint64_t)std::max(1, v.sm_count / (int)kSmsPerPair));
    rc = i8_launch(h, v.functions[p.index], grid, I8_PAIR_THREADS, i8_function_smem(p.index, v.main_smem), 0, stream, params);
    i8_note(h, p.index == kHalf ? 4 : 1, 1, grid, tile_n);
    return rc;
}

SGEMM_API int sgemm_i8_quantize(sgemm_handle *h, const void *dX, int x_type, int8_t *dQ, float *dScale, uint32_t k, uint32_t n,
                                uint32_t ldx, uint32_t ldq, int pow2, void *stream) {
    const char *op = "sgemm_i8_quantize";
    I8View v;
    int rc = begin(h, op, &v);
    if (rc) return rc;
    if (!known_type(x_type)) return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "X's type is FP32 (0), FP16 (1) or BF16 (2)");
    if (pow2 != 0 && pow2 != 1) return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "pow2 is 0 (scale max/127) or 1 (power of two)");
    if (ldx < std::max(k, 1u) || ldq < std::max(k, 1u))
        return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "a leading dimension is smaller than the rows it must hold");
    if (n == 0) return SGEMM_OK;
    if (k > kLongestRow || n > kLargest) return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "problem too large");
    if (!dScale || (k && (!dX || !dQ))) return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "X, Q or the scales are NULL");
    const uint32_t eb = type_bytes(x_type);
    if (!aligned(dX, eb) || !aligned(dScale, 4)) return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "X or the scales are not aligned to their element type");
    RowArgs a{dX, nullptr, nullptr, nullptr, dQ, dScale, k, n, ldx, 0, 0, ldq, 32, 0, 0, (uint32_t)pow2, 0.0f, 0.0f};
    return launch_rows(h, v, kQuantize, x_type, a, stream);
}

SGEMM_API int sgemm_i8_restore(sgemm_handle *h, const int8_t *dQ, const float *dScale, void *dOut, int out_type, uint32_t k,
                               uint32_t n, uint32_t ldq, uint32_t ldo, void *stream) {
    const char *op = "sgemm_i8_restore";
    I8View v;
    int rc = begin(h, op, &v);
    if (rc) return rc;
    if (!known_type(out_type)) return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "the output's type is FP32 (0), FP16 (1) or BF16 (2)");
    if (ldq < std::max(k, 1u) || ldo < std::max(k, 1u))
        return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "a leading dimension is smaller than the rows it must hold");
    if (n == 0 || k == 0) return SGEMM_OK;
    if (k > kLargest || n > kLargest) return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "problem too large");
    if (!dQ || !dScale || !dOut) return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "Q, the scales or the output are NULL");
    const uint32_t eb = type_bytes(out_type);
    if (!aligned(dOut, eb) || !aligned(dScale, 4)) return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "the output or the scales are not aligned to their element type");
    const bool vec = aligned(dQ, 16) && ldq % 16 == 0 && aligned(dOut, 16) && (uint64_t)ldo * eb % 16 == 0;
    const uint64_t units = (uint64_t)(vec ? ceil_div(k, 16) : ceil_div(k, 16 / eb) + 1) * n;
    const uint32_t blocks = (uint32_t)std::min<uint64_t>((units + 255) / 256, (uint64_t)v.sm_count * 32);
    I8Scope scope(h);
    void *params[] = {&dQ, &dScale, &dOut, &k, &n, &ldq, &ldo};
    return i8_launch(h, v.functions[kRestore + 2 * out_type + (vec ? 0 : 1)], blocks, 256, 0, 0, stream, params);
}

SGEMM_API int sgemm_i8_rmsnorm(sgemm_handle *h, const void *dX, const void *dResidual, const void *dGamma, int x_type, float eps,
                               int8_t *dQ, float *dScale, void *dSum, uint32_t k, uint32_t n, uint32_t ldx, uint32_t ldr,
                               uint32_t ldq, uint32_t lds, void *stream) {
    const char *op = "sgemm_i8_rmsnorm";
    I8View v;
    int rc = begin(h, op, &v);
    if (rc) return rc;
    if (!known_type(x_type)) return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "X's type is FP32 (0), FP16 (1) or BF16 (2)");
    if (!(eps >= 0.0f) || eps > 3.0e38f) return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "eps must be a finite number that is not negative");
    if (k == 0) return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "K = 0: the mean of no squares is not defined");
    if (ldx < k || ldq < k || (dResidual && ldr < k) || (dSum && lds < k))
        return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "a leading dimension is smaller than the rows it must hold");
    if (n == 0) return SGEMM_OK;
    if (k > kLongestRow || n > kLargest) return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "problem too large");
    if (!dX || !dGamma || !dQ || !dScale) return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "X, gamma, Q or the scales are NULL");
    const uint32_t eb = type_bytes(x_type);
    if (!aligned(dX, eb) || !aligned(dGamma, eb) || !aligned(dResidual, eb) || !aligned(dSum, eb) || !aligned(dScale, 4))
        return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "a matrix is not aligned to its element type");
    if ((dSum == dX && dX && lds != ldx) || (dSum == dResidual && dSum && lds != ldr))
        return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "the sum may replace X or the residual only with the same leading dimension");
    RowArgs a{dX, dResidual, dGamma, dSum, dQ, dScale, k, n, ldx, ldr, lds, ldq, 32, 0, 0, 0, eps, 0.0f};
    return launch_rows(h, v, kNorm, x_type, a, stream);
}

SGEMM_API int sgemm_i8_wgrad(sgemm_handle *h, const int8_t *dQ, const float *dScale, const void *dG, int g_type, const void *dC,
                             void *dD, int d_type, float alpha, float beta, uint32_t m, uint32_t n, uint32_t tokens,
                             uint32_t ldq, uint32_t ldg, uint32_t ldc, uint32_t ldd, void *stream) {
    const char *op = "sgemm_i8_wgrad";
    I8View v;
    int rc = begin(h, op, &v);
    if (rc) return rc;
    if (g_type != (int)SGEMM_I8_FP16 && g_type != (int)SGEMM_I8_BF16) return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "G's type is FP16 (1) or BF16 (2)");
    if (!known_type(d_type)) return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "D's type is FP32 (0), FP16 (1) or BF16 (2)");
    if (ldq < std::max(m, 1u) || ldg < std::max(n, 1u) || ldd < std::max(m, 1u) || (beta != 0.0f && ldc < std::max(m, 1u)))
        return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "a leading dimension is smaller than the rows it must hold");
    if (m == 0 || n == 0) return SGEMM_OK;
    if (m > kLargest || n > kLargest || tokens > kLargest) return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "problem too large");
    if (!dD || (tokens && (!dQ || !dScale || !dG))) return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "D, the checkpoint, its scales or G are NULL");
    if (beta != 0.0f && !dC) return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "C is NULL but beta != 0");
    if (beta != 0.0f && dC == dD && ldc != ldd)
        return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "D may replace C only with the same leading dimension");
    if (!aligned(dG, 2) || !aligned(dScale, 4) || !aligned(dD, type_bytes(d_type)) || (beta != 0.0f && !aligned(dC, type_bytes(d_type))))
        return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "a matrix is not aligned to its element type");
    const bool tma = aligned(dQ, 16) && ldq % 16 == 0 && aligned(dG, 16) && ldg % 8 == 0 && tokens > 0;
    if (v.force_variant != 0 && v.force_variant != 2 && !tma)
        return refuse(h, SGEMM_ERR_UNSUPPORTED, op, "the tensor kernel is forced but the operands need 16-byte aligned bases, ldq a multiple of 16, ldg of 8, and a token");
    I8Scope scope(h);
    WgradArgs a{dQ, dScale, dG, dC, dD, v.status, m, n, tokens, ldq, ldg, ldc, ldd, (uint32_t)g_type, (uint32_t)d_type, alpha, beta, 0, 0};
    if (!tma || v.force_variant == 2) {
        a.tiles_m = ceil_div(m, I8_SIMT_TILE);
        a.tiles_n = ceil_div(n, I8_SIMT_TILE);
        const uint64_t tiles = (uint64_t)a.tiles_m * a.tiles_n;
        if (tiles > 0x7FFFFFFFull) return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "problem too large");
        void *params[] = {&a};
        rc = i8_launch(h, v.functions[kWgradSimt], (uint32_t)tiles, I8_SIMT_THREADS, 0, 0, stream, params);
        i8_note(h, 2, 1, (uint32_t)tiles, I8_SIMT_TILE);
        return rc;
    }
    a.tiles_m = ceil_div(m, 256);
    a.tiles_n = ceil_div(n, 256);
    const uint64_t tiles = (uint64_t)a.tiles_m * a.tiles_n;
    if (tiles > 0x3FFFFFFFull) return refuse(h, SGEMM_ERR_INVALID_ARGUMENT, op, "problem too large");
    const uint32_t pairs = (uint32_t)std::max(1, v.sm_count / (int)kSmsPerPair), stages = ceil_div(tokens, I8W_BK);
    // Too few tiles for the device: cut the tokens into as many parts (up to 4) as still run at the same time, with at least eight
    // stages each.  (Clusters do not fill the device: 74 of 2 CTAs, but 33 of 4, 22 of 6 and 15 of 8 fit the
    // 148 SMs with their uneven groups, and one cluster too many is a second wave: 16 tiles over 16384 tokens
    // take 62 us in 2 parts and 71 in 4.)
    uint32_t parts = 1;
    for (uint32_t p = 2; p <= 4; ++p)
        if (tiles <= v.wgrad_clusters[p] && stages >= p * 8) parts = p;
    if (v.split_k > 0) parts = (uint32_t)std::min<int64_t>(v.split_k, 4);
    parts = std::min(parts, stages);
    const uint32_t units = parts > 1 ? (uint32_t)tiles : (uint32_t)std::min<uint64_t>(tiles, pairs);
    const uint32_t grid = units * 2 * parts;
    I8TensorMap map_q, map_g;
    if ((rc = i8_encode(h, &map_q, kMapInt8, dQ, m, tokens, ldq, 128, I8W_BK, false))) return rc;
    if ((rc = i8_encode(h, &map_g, g_type == (int)SGEMM_I8_BF16 ? kMapBf16 : kMapFp16, dG, n, tokens, (uint64_t)ldg * 2, 64, I8W_BK, true))) return rc;
    void *params[] = {&a, &map_q, &map_g};
    rc = i8_launch(h, v.functions[kWgrad], grid, I8W_THREADS, I8W_SMEM, 2 * parts, stream, params);
    i8_note(h, 1, parts, grid, 256);
    return rc;
}
