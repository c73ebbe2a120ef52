// ---------------------------------------------------------------------------------------------
// Row kernels of the 8-bit operators.  A "row" is one column of a column-major K x N matrix: K contiguous elements, one
// token or one output channel.
//
//   quantize   P = max |x|
//              finest scale:       s = P / 127,                  q = round(127 x / P)
//              power of two:       s = least 2^e >= P / 127,      q = round(x / s)
//   rmsnorm    h = x + r (FP32; also stored, rounded to x's type),  p = h * g (FP32),  P = max |p|
//              s = P / 127 * rsqrt(mean h^2 + eps),              q = round(127 p / P)
//   restore    x = s * q, rounded to the output's type
//
// round() goes to the nearest integer, halves to the even one, of the EXACT quotient.  The norm's rsqrt scales a whole row
// and leaves 127 p / P alone, so q depends on no sum and on no order of one: every element of q is a function of x, r
// and g that a host can restate bit for bit.  FP32 gives the quotient to 2^-24 of its value (below 127: within 8e-6), and
// the few elements nearer than 1e-5 to a half (two in 10^5) are decided by comparing 127 |p| with (n + 1/2) P in FP64,
// where both products are exact.  A power-of-two scale makes x / s exact and needs no such step; it is what
// activation checkpoints want, because s * q then has at most 7 significant bits and is exact in FP16 and BF16.
//
// A row of zeros gets s = 0 and q = 0.  A row that holds a NaN, an infinity, or a value beyond 127 * 2^121 (restoring it
// could overflow) gets s = NaN and q = 0: what is computed from it is NaN, rather than a finite number that is wrong.
//
// What bounds them: memory.  A row is read once and stays in registers between the reduction and the rounding (NV vectors of 16 bytes
// per thread; rows too long for that are read twice).  `tpr` threads work on a row, several rows share a block when they
// are short, and the blocks of an SM are at different stages, so loads, reductions and stores overlap.
// The arithmetic is kept below the issue rate that memory leaves (about 16 instructions an element at 6.5 TB/s):
// int8 and the integer part of a float change places through the mantissa of 1.5 * 2^23, not the conversion unit.
// ---------------------------------------------------------------------------------------------
#define I8_ROUND_MAGIC 12582912.0f          // 1.5 * 2^23: adding it rounds to the nearest integer, into the low mantissa bits
#define I8_LARGEST_BITS 0x7F7E0000u         // 127 * 2^121 as an FP32 word

struct I8RowArgs {
    const void *x;
    const void *r;        // norm: residual added to x, or NULL
    const void *g;        // norm: weights of the K features
    void *sum;            // norm: x + r rounded to x's type, or NULL (may be r or x itself)
    int8_t *q;
    float *scale;
    uint32_t k, rows, ldx, ldr, lds, ldq;
    uint32_t tpr;         // threads per row, a power of two, 32 .. 1024
    uint32_t pow2;
    float eps;
};

__device__ __forceinline__ uint32_t i8_abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// round(127 |p| / P) for a quotient that lies next to n + 1/2: both sides of the comparison are exact in FP64
// (24 + 7 and 24 + 8 significant bits).
__device__ __noinline__ int i8_round_exact(float p, float peak, float quotient) {
    const int n = (int)floorf(fabsf(quotient));
    const double a = 127.0 * fabs((double)p), b = ((double)n + 0.5) * (double)peak;
    const int up = a > b ? 1 : a < b ? 0 : (n & 1);
    return p < 0.0f ? -(n + up) : n + up;
}

template <uint32_t TYPE, int NV, bool NORM, bool VEC>
__device__ __forceinline__ void i8_rows_body(const I8RowArgs &a) {
    using E = I8Elem<TYPE>;
    using T = typename E::type;
    constexpr int VE = 16 / (int)sizeof(T);   // elements of a 16-byte vector
    constexpr int PER = NV * VE;              // elements a thread keeps
    __shared__ float red_sum[32], red_small[32];
    __shared__ uint32_t red_max[32];

    sgemm_launch_dependents();
    sgemm_grid_dependency_wait();
    const uint32_t rows_per_block = blockDim.x / a.tpr;
    const uint32_t row = blockIdx.x * rows_per_block + threadIdx.x / a.tpr;
    const uint32_t t = threadIdx.x & (a.tpr - 1);
    const bool live = row < a.rows;
    const T *x = static_cast<const T *>(a.x) + (uint64_t)(live ? row : 0) * a.ldx;
    const T *r = NORM && a.r ? static_cast<const T *>(a.r) + (uint64_t)(live ? row : 0) * a.ldr : nullptr;
    const T *g = static_cast<const T *>(a.g);
    T *sum = NORM && a.sum ? static_cast<T *>(a.sum) + (uint64_t)(live ? row : 0) * a.lds : nullptr;
    int8_t *q = a.q + (uint64_t)(live ? row : 0) * a.ldq;
    const uint32_t k = live ? a.k : 0u;
    const uint32_t span = a.tpr * PER;        // elements of a row one pass covers
    const uint32_t passes = a.k ? (a.k + span - 1) / span : 1u;

    // VEC: a thread's elements are vectors, t-th of every tpr; otherwise single elements, t-th of every tpr
    auto index = [&](uint32_t pass, int i, int j) -> uint32_t {
        return VEC ? pass * span + (i * a.tpr + t) * VE + j : pass * span + (i * VE + j) * a.tpr + t;
    };
    float p[PER];
    float squares = 0.0f, squares_small = 0.0f;   // of h and of h * 2^-64 (for rows whose squares leave FP32)
    uint32_t peak_bits = 0u;

    auto load = [&](const T *src, uint32_t pass, int i, float (&v)[VE]) {
        if (VEC) {
            const uint32_t e = index(pass, i, 0);
            if (e + VE <= k) {
                const uint4 w = *reinterpret_cast<const uint4 *>(src + e);
                const T *pv = reinterpret_cast<const T *>(&w);
#pragma unroll
                for (int j = 0; j < VE; ++j) v[j] = E::get(pv[j]);
                return;
            }
        }
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            const uint32_t e = index(pass, i, j);
            v[j] = e < k ? E::get(src[e]) : 0.0f;
        }
    };
    auto fetch = [&](uint32_t pass, bool store_sum) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float v[VE];
            load(x, pass, i, v);
            if (NORM) {
                if (r) {
                    float w[VE];
                    load(r, pass, i, w);
#pragma unroll
                    for (int j = 0; j < VE; ++j) v[j] = __fadd_rn(v[j], w[j]);
                }
                if (sum && store_sum) {
                    const uint32_t e = index(pass, i, 0);
                    if (VEC && e + VE <= k) {
                        uint4 w;
                        T *pw = reinterpret_cast<T *>(&w);
#pragma unroll
                        for (int j = 0; j < VE; ++j) pw[j] = E::put(v[j]);
                        *reinterpret_cast<uint4 *>(sum + e) = w;
                    } else {
#pragma unroll
                        for (int j = 0; j < VE; ++j)
                            if (index(pass, i, j) < k) sum[index(pass, i, j)] = E::put(v[j]);
                    }
                }
                float w[VE];
                load(g, pass, i, w);
#pragma unroll
                for (int j = 0; j < VE; ++j) {
                    squares = fmaf(v[j], v[j], squares);
                    if (TYPE != SGEMM_I8_FP16) {   // (sums of FP16 pairs cannot leave FP32 when squared)
                        const float small = v[j] * 0x1p-64f;
                        squares_small = fmaf(small, small, squares_small);
                    }
                    v[j] = __fmul_rn(v[j], w[j]);
                }
            }
#pragma unroll
            for (int j = 0; j < VE; ++j) p[i * VE + j] = v[j];
        }
    };
    auto track = [&] {
#pragma unroll
        for (int j = 0; j < PER; ++j) peak_bits = max(peak_bits, i8_abs_bits(p[j]));   // as integers NaN > infinity > finite
    };
    fetch(0, passes == 1);
    track();
    for (uint32_t pass = 1; pass < passes; ++pass) {
        fetch(pass, false);
        track();
    }

    // the row's largest magnitude and its sum of squares, in a fixed order
    peak_bits = __reduce_max_sync(0xffffffffu, peak_bits);
    if (NORM) {
#pragma unroll
        for (int d = 16; d; d >>= 1) {
            squares += __shfl_xor_sync(0xffffffffu, squares, d);
            if (TYPE != SGEMM_I8_FP16) squares_small += __shfl_xor_sync(0xffffffffu, squares_small, d);
        }
    }
    if (a.tpr > 32) {
        const uint32_t warp = threadIdx.x >> 5, warps = a.tpr >> 5, first = warp & ~(warps - 1);
        if ((threadIdx.x & 31) == 0) {
            red_max[warp] = peak_bits;
            if (NORM) {
                red_sum[warp] = squares;
                red_small[warp] = squares_small;
            }
        }
        __syncthreads();
        const uint32_t lane = threadIdx.x & 31;
        const bool mine = lane < warps;
        peak_bits = __reduce_max_sync(0xffffffffu, mine ? red_max[first + lane] : 0u);
        if (NORM) {
            squares = mine ? red_sum[first + lane] : 0.0f;
            squares_small = mine ? red_small[first + lane] : 0.0f;
#pragma unroll
            for (int d = 16; d; d >>= 1) {
                squares += __shfl_xor_sync(0xffffffffu, squares, d);
                if (TYPE != SGEMM_I8_FP16) squares_small += __shfl_xor_sync(0xffffffffu, squares_small, d);
            }
        }
    }
    if (!live) return;

    float peak = __uint_as_float(peak_bits), lift = 1.0f, scale, inverse;
    const bool bad = peak_bits > I8_LARGEST_BITS, zero = peak_bits == 0u;
    if (a.pow2) {
        // P = m 2^e: 127 * 2^(e-6) holds it up to m = 127/64, else 2^(e-5); subnormal scales are avoided
        const int e = max((int)(peak_bits >> 23) - 127 - ((peak_bits & 0x7FFFFFu) <= 0x7E0000u ? 6 : 5), -126);
        scale = __uint_as_float((uint32_t)(e + 127) << 23);
        inverse = __uint_as_float((uint32_t)(127 - e) << 23);
    } else {
        scale = __fdiv_rn(peak, 127.0f);
        if (peak < 0x1p-100f) {   // 127 / P must not overflow
            lift = 0x1p64f;
            peak *= lift;
        }
        inverse = __fdiv_rn(127.0f, peak);
    }
    if (NORM) {
        const float mean = __fdiv_rn(squares, (float)a.k);
        float rstd = __frcp_rn(__fsqrt_rn(mean + a.eps));
        if (TYPE != SGEMM_I8_FP16 && !(squares < INFINITY)) rstd = 0x1p-64f * __frcp_rn(__fsqrt_rn(__fdiv_rn(squares_small, (float)a.k)));
        scale *= rstd;
    }
    if (zero) { scale = 0.0f; inverse = 0.0f; lift = 0.0f; }
    if (bad) scale = __uint_as_float(0x7FFFFFFFu);
    if (t == 0) a.scale[row] = scale;

    for (uint32_t pass = 0; pass < passes; ++pass) {
        if (passes > 1) fetch(pass, true);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            uint32_t word[VE / 4];
            float worst = 0.0f;
#pragma unroll
            for (int w = 0; w < VE / 4; ++w) {
                uint32_t b[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float v = lift == 1.0f ? p[i * VE + w * 4 + j] : p[i * VE + w * 4 + j] * lift;
                    const float f = fmaf(v, inverse, I8_ROUND_MAGIC);
                    worst = fmaxf(worst, fabsf(fmaf(v, inverse, -(f - I8_ROUND_MAGIC))));
                    b[j] = __float_as_uint(f);
                }
                word[w] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
            }
            if (worst > 0.49999f && !a.pow2 && !bad) {
#pragma unroll
                for (int w = 0; w < VE / 4; ++w)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float v = p[i * VE + w * 4 + j] * lift;
                        const float f = fmaf(v, inverse, I8_ROUND_MAGIC);
                        if (fabsf(fmaf(v, inverse, -(f - I8_ROUND_MAGIC))) > 0.49999f) {
                            const uint32_t byte = (uint32_t)i8_round_exact(v, peak, v * inverse) & 0xFFu;
                            word[w] = (word[w] & ~(0xFFu << (8 * j))) | (byte << (8 * j));
                        }
                    }
            }
            if (bad) {
#pragma unroll
                for (int w = 0; w < VE / 4; ++w) word[w] = 0u;
            }
            const uint32_t e = index(pass, i, 0);
            if (VEC && e + VE <= k) {
                if constexpr (VE == 8) *reinterpret_cast<uint2 *>(q + e) = make_uint2(word[0], word[1]);
                else *reinterpret_cast<uint32_t *>(q + e) = word[0];
            } else {
#pragma unroll
                for (int j = 0; j < VE; ++j)
                    if (index(pass, i, j) < k) q[index(pass, i, j)] = (int8_t)(word[j / 4] >> (8 * (j & 3)));
            }
        }
    }
}

// One kernel per element type, vectors kept per thread and access form; the host picks by K, alignment and row count.
#define I8_ROW_KERNEL(NAME, TYPE, NV, NORM, VEC)                                                          \
    extern "C" __global__ void __launch_bounds__(I8_ROW_MAX_THREADS) NAME(const __grid_constant__ I8RowArgs a) { \
        i8_rows_body<TYPE, NV, NORM, VEC>(a);                                                             \
    }
#define I8_ROW_KERNELS(OP, NORM, NAME, TYPE)             \
    I8_ROW_KERNEL(OP##_##NAME##_v1, TYPE, 1, NORM, true) \
    I8_ROW_KERNEL(OP##_##NAME##_v2, TYPE, 2, NORM, true) \
    I8_ROW_KERNEL(OP##_##NAME##_v4, TYPE, 4, NORM, true) \
    I8_ROW_KERNEL(OP##_##NAME##_s4, TYPE, 4, NORM, false)
I8_ROW_KERNELS(i8_quantize, false, fp32, SGEMM_I8_FP32)
I8_ROW_KERNELS(i8_quantize, false, fp16, SGEMM_I8_FP16)
I8_ROW_KERNELS(i8_quantize, false, bf16, SGEMM_I8_BF16)
I8_ROW_KERNELS(i8_rmsnorm, true, fp32, SGEMM_I8_FP32)
I8_ROW_KERNELS(i8_rmsnorm, true, fp16, SGEMM_I8_FP16)
I8_ROW_KERNELS(i8_rmsnorm, true, bf16, SGEMM_I8_BF16)

// ---------------------------------------------------------------------------------------------
// restore: every thread widens 16 consecutive int8 of a row (VEC) or one (operands that are not aligned).
// ---------------------------------------------------------------------------------------------
template <uint32_t TYPE, bool VEC>
__device__ __forceinline__ void i8_restore_body(const int8_t *q, const float *scale, void *out, uint32_t k, uint32_t rows,
                                                uint32_t ldq, uint32_t ldo) {
    using E = I8Elem<TYPE>;
    using T = typename E::type;
    sgemm_launch_dependents();
    sgemm_grid_dependency_wait();
    constexpr uint32_t STEP = VEC ? 16 : 1;
    const uint32_t units = (k + STEP - 1) / STEP;   // of a row
    const uint64_t total = (uint64_t)units * rows, stride = (uint64_t)gridDim.x * blockDim.x;
    for (uint64_t at = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; at < total; at += stride) {
        const uint32_t row = total <= 0xFFFFFFFFull ? (uint32_t)at / units : (uint32_t)(at / units);
        const uint32_t e = (uint32_t)(at - (uint64_t)row * units) * STEP;
        const float s = scale[row];
        const int8_t *src = q + (uint64_t)row * ldq + e;
        T *dst = static_cast<T *>(out) + (uint64_t)row * ldo + e;
        if (VEC && e + 16 <= k) {
            const uint4 w = *reinterpret_cast<const uint4 *>(src);
            const uint32_t words[4] = {w.x, w.y, w.z, w.w};
            uint4 o[sizeof(T)];
            T *po = reinterpret_cast<T *>(o);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v[4];
                i8_widen4(words[i], v);
#pragma unroll
                for (int j = 0; j < 4; ++j) po[4 * i + j] = E::put(v[j] * s);
            }
#pragma unroll
            for (int i = 0; i < (int)sizeof(T); ++i) reinterpret_cast<uint4 *>(dst)[i] = o[i];
        } else {
            for (uint32_t j = 0; j < STEP && e + j < k; ++j) dst[j] = E::put((float)src[j] * s);
        }
    }
}
#define I8_RESTORE_KERNEL(NAME, TYPE, VEC)                                                                              \
    extern "C" __global__ void __launch_bounds__(256) NAME(const int8_t *q, const float *scale, void *out, uint32_t k, \
                                                           uint32_t rows, uint32_t ldq, uint32_t ldo) {                \
        i8_restore_body<TYPE, VEC>(q, scale, out, k, rows, ldq, ldo);                                                  \
    }
I8_RESTORE_KERNEL(i8_restore_fp32_v, SGEMM_I8_FP32, true)
I8_RESTORE_KERNEL(i8_restore_fp16_v, SGEMM_I8_FP16, true)
I8_RESTORE_KERNEL(i8_restore_bf16_v, SGEMM_I8_BF16, true)
I8_RESTORE_KERNEL(i8_restore_fp32_s, SGEMM_I8_FP32, false)
I8_RESTORE_KERNEL(i8_restore_fp16_s, SGEMM_I8_FP16, false)
I8_RESTORE_KERNEL(i8_restore_bf16_s, SGEMM_I8_BF16, false)
