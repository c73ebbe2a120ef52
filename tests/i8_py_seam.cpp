// Stand-in for the library behind the Python binding (csrc/sgemm_py.cpp is compiled with this file in place of libsgemm_runner.so): the calls
// note their arguments and can be made to wait for a flag, as a launch waits for room in a full queue.
#include "sgemm_runner.h"

#include <chrono>
#include <thread>

extern "C" {
__attribute__((visibility("default"))) volatile int seam_wait = 0, seam_flag = 0, seam_calls = 0;
__attribute__((visibility("default"))) uint32_t seam_ld[4];   // the leading dimensions of the last call, in the order of its arguments
}

namespace {
int answer(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    ++seam_calls;
    seam_ld[0] = a; seam_ld[1] = b; seam_ld[2] = c; seam_ld[3] = d;
    const auto limit = std::chrono::steady_clock::now() + std::chrono::seconds(3);
    while (seam_wait && !seam_flag) {
        if (std::chrono::steady_clock::now() > limit) return -77;
        std::this_thread::sleep_for(std::chrono::milliseconds(1));
    }
    return 0;
}
}  // namespace

extern "C" {
int sgemm_i8_linear(sgemm_handle *, const int8_t *, const float *, const int8_t *, const float *, const float *, void *, int, uint32_t, uint32_t,
                    uint32_t, uint32_t ldw, uint32_t ldx, uint32_t ldy, void *) { return answer(ldw, ldx, ldy, 0); }
int sgemm_i8_quantize(sgemm_handle *, const void *, int, int8_t *, float *, uint32_t, uint32_t, uint32_t ldx, uint32_t ldq, int, void *) {
    return answer(ldx, ldq, 0, 0);
}
int sgemm_i8_restore(sgemm_handle *, const int8_t *, const float *, void *, int, uint32_t, uint32_t, uint32_t ldq, uint32_t ldo, void *) {
    return answer(ldq, ldo, 0, 0);
}
int sgemm_i8_rmsnorm(sgemm_handle *, const void *, const void *, const void *, int, float, int8_t *, float *, void *, uint32_t, uint32_t,
                     uint32_t ldx, uint32_t ldr, uint32_t ldq, uint32_t lds, void *) { return answer(ldx, ldr, ldq, lds); }
int sgemm_i8_wgrad(sgemm_handle *, const int8_t *, const float *, const void *, int, const void *, void *, int, float, float, uint32_t, uint32_t,
                   uint32_t, uint32_t ldq, uint32_t ldg, uint32_t ldc, uint32_t ldd, void *) { return answer(ldq, ldg, ldc, ldd); }
}
