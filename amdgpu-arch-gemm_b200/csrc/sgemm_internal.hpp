// Internal seam between the translation units of libsgemm_runner.so (not part of the C ABI).
#pragma once
#include "sgemm_runner.h"

#include <cstddef>
#include <cstdint>

namespace sgemm_internal {

// Device ordinal the handle was opened on.
int handle_device(const sgemm_handle *h);

// Record a failure message on the handle (what sgemm_last_error returns) and hand `code` back.
int set_error(sgemm_handle *h, int code, const char *message);

// Scratch bytes sgemm_launch would need for this problem under the handle's current options, planned for the
// operands the call will really get (a base TMA cannot read where it lies adds an aligned copy to the need).
int scratch_bytes(sgemm_handle *h, const void *dA, const void *dB, uint32_t m, uint32_t n, uint32_t k, uint32_t lda,
                  uint32_t ldb, size_t *bytes);

// Run `fn(arg)` with the handle's CUDA context current on this thread (pushed before, popped after), so that
// CUDA runtime calls made inside bind to the device the handle was opened on without cudaSetDevice.  Returns
// what `fn` returns, or SGEMM_ERR_CUDA when the context cannot be made current.
int with_context(sgemm_handle *h, int (*fn)(void *), void *arg);

// One pointer-sized slot per handle for sgemm_noalloc.cu: the device address of the library's static scratch
// array as resolved in the handle's context (NULL until the first allocation-free call on the handle).
void **noalloc_scratch_slot(sgemm_handle *h);

// The handle's communicator over the GPUs that share one sharded SGEMM (sgemm_multi.cpp owns the NCCL side):
// `comm` is an ncclComm_t, NULL until sgemm_comm_init / sgemm_comm_init_all.
struct CommState {
    void *comm = nullptr;
    int rank = 0;
    int world = 1;
};
CommState *comm_state(sgemm_handle *h);

// In-place exchange over the handle's communicator, ordered on `stream`: piece r — `bytes[r]` bytes at
// `base + offsets[r]` on every rank, valid on rank r — is copied to the same place on all other ranks.  Equal,
// back-to-back pieces go as one all-gather, ragged ones as grouped broadcasts.
int comm_complete(sgemm_handle *h, void *base, const size_t *offsets, const size_t *bytes, void *stream);

// Destroy an ncclComm_t stored in a CommState (no-op for NULL or without NCCL).
void comm_release(void *comm);

// sgemm_launch with the scratch taken from [scratch, scratch + scratch_bytes) for this one call only; the
// handle's own workspace settings are put back before returning.  Never allocates device memory; a need beyond
// `scratch_bytes` comes back as SGEMM_ERR_SCRATCH_LIMIT.
int launch_with_scratch(sgemm_handle *h, void *scratch, size_t scratch_bytes, const float *dA, const float *dB,
                        const float *dC, float *dD, float alpha, float beta, uint32_t m, uint32_t n, uint32_t k,
                        uint32_t lda, uint32_t ldb, uint32_t ldc, uint32_t ldd, void *stream);

// ---- seam of the 8-bit entry points (sgemm_i8.cpp) ----------------------------------------------------------------
// A CUDA tensor map as plain bytes (the host code of the entry points needs no <cuda.h>).
struct alignas(64) I8TensorMap {
    uint64_t opaque[16];
};
constexpr int kI8Functions = 64;
// What the planner needs to know about a handle of an INT8 cubin.
struct I8View {
    void *const *functions = nullptr;   // kernels by index (sgemm_i8.cpp numbers and names them)
    uint32_t *status = nullptr;         // device status words
    int sm_count = 0;
    uint32_t tile_n = 0, main_smem = 0;   // the main linear kernel as generated
    int64_t force_variant = 0, split_k = 0;                 // options of sgemm_set_option
    uint32_t wgrad_clusters[5] = {0, 0, 0, 0, 0};           // clusters of 2 * i CTAs of the weight gradient the device holds at a time
};
// False when the handle's cubin was not generated for INT8 operands.
bool i8_view(sgemm_handle *h, I8View *view);
// The kernels sgemm_open resolves in an INT8 cubin: their names, the dynamic shared memory they opt in to, and, where a
// kernel hands registers from one warp group to another, the registers per thread it must have been compiled to (else 0).
int i8_function_count();
const char *i8_function_name(int index);
uint32_t i8_function_smem(int index, uint32_t main_smem);
int i8_function_registers(int index);
int i8_wgrad_function();   // index of the weight gradient's kernel, and its block size
uint32_t i8_wgrad_threads();
// The words an INT8 cubin carries as `sgemm_i8_layout` when it was compiled from the sources of this library.
const uint32_t *i8_layout(size_t *words);
// Make the handle's context current on this thread for the object's life (tensor maps and launches need one; the caller's is put back).
class I8Scope {
public:
    explicit I8Scope(sgemm_handle *h);
    ~I8Scope();
    I8Scope(const I8Scope &) = delete;
    I8Scope &operator=(const I8Scope &) = delete;

private:
    bool pushed_ = false;
};
// Launch (inside an I8Scope); cluster: CTAs per cluster (0: as compiled).
int i8_launch(sgemm_handle *h, void *function, uint32_t grid, uint32_t threads, uint32_t smem, uint32_t cluster, void *stream,
              void **params);
// 2-D tensor map (inside an I8Scope), dims {d0 (contiguous), d1}, box {b0, b1}, with the 128-byte swizzle or none.
enum I8MapType { kMapInt8, kMapFp16, kMapBf16 };
int i8_encode(sgemm_handle *h, I8TensorMap *map, I8MapType type, const void *base, uint64_t d0, uint64_t d1, uint64_t stride_bytes,
              uint32_t b0, uint32_t b1, bool swizzle);
// What sgemm_get_info reports as "last_variant", "last_split_k", "last_grid" and "last_tile_n".
void i8_note(sgemm_handle *h, int variant, uint32_t parts, uint32_t grid, uint32_t tile_n);

}  // namespace sgemm_internal
