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
// and g that a host can restate bit for bit.  FP32 gives the quotient to 2^-15.4; the elements nearer than 2^-14 to a half (12 in
// 10^5) are decided by the quotient in FP64 (127 p is exact there, and no quotient of FP32 numbers that is not a tie
// comes closer to one than FP64 tells apart).  A power-of-two scale makes x / s exact and needs no such step; it is what
// activation checkpoints want, because s * q then has at most 7 significant bits and is exact in FP16 and BF16.
//
// A row of zeros gets s = 0 and q = 0.  A row that holds a NaN, an infinity, or a value beyond 127 * 2^121 (restoring it
// could overflow) gets s = NaN and q = 0: what is computed from it is NaN, rather than a finite number that is wrong.
//
// What bounds them: memory.  A row is read once and stays in registers between the reduction and the rounding, PER = 8, 16 or 32
// elements per thread (rows longer than 8192 are read twice).  `tpr` threads work on a row, several rows share a block when
// they are short, and the blocks of an SM are at different stages, so loads, reductions and stores overlap.  All loads of a
// row come before its first store: the sum may lie over the residual, so the compiler cannot move a load across a store itself.
// The arithmetic is kept below the issue rate that memory leaves (about 16 instructions an element at 6.5 TB/s for quantize):
// int8 and the integer part of a float change places through the mantissa, not the conversion unit, and the row's peak is
// taken on packed 16-bit pairs.
// ---------------------------------------------------------------------------------------------
#define I8_ROUND_MAGIC 12582912.0f          // 1.5 * 2^23: adding it rounds to the nearest integer, into the low mantissa bits
#define I8_LARGEST_BITS 0x7F7E0000u         // 127 * 2^121 as an FP32 word
#define I8_TINY 0x1p-100f                   // peaks below it: 127 / P is not formed in FP32
// Rows whose squares leave FP32 have a second sum, of (h * 2^-96)^2.  Of the largest FP32 number that is below 2^64, so the longest row's
// (2^30) stays below 2^94; and where the plain sum passed 2^128, squares that matter to 2^-24 of it were above 2^74, here 2^-118.
#define I8_DOWN 0x1p-96f
// Where neither the plain sum nor eps reaches 2^-90, squares may vanish: a third sum, of (h * 2^92)^2, stays below 2^94 there, and the square of
// the smallest FP32 number is 2^-114 in it.  (A plain sum of at least 2^-90 lacks at most 2^30 * 2^-150.)
#define I8_FAINT 0x1p-90f
#define I8_UP 0x1p92f

struct I8RowArgs {
    const void *x;
    const void *r;        // norm: residual added to x, or NULL
    const void *g;        // norm: weights of the K features
    void *sum;            // norm: x + r rounded to x's type, or NULL (may be r or x itself)
    int8_t *q;
    float *scale;
    uint32_t k, rows, ldx, ldr, lds, ldq;
    uint32_t tpr;         // threads per row, a power of two, 32 .. 1024 (PER 8), 512 (16) or 256 (32)
    uint32_t tpr_log2, passes;   // how often tpr * PER elements take a row (host: an integer division is 30 instructions)
    uint32_t pow2;
    float eps, inv_k;
};

__device__ __forceinline__ uint32_t i8_abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// max that hands a NaN on (the operands are not negative)
__device__ __forceinline__ float i8_max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// The elements of a 16-byte vector, and back.
template <uint32_t TYPE>
__device__ __forceinline__ void i8_unpack2(uint32_t w, float &lo, float &hi) {
    if (TYPE == SGEMM_I8_BF16) {
        lo = __uint_as_float(w << 16);
        hi = __uint_as_float(w & 0xFFFF0000u);
    } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
        lo = f.x;
        hi = f.y;
    }
}
template <uint32_t TYPE>
__device__ __forceinline__ uint32_t i8_pack2(float lo, float hi) {
    uint32_t w;
    if (TYPE == SGEMM_I8_BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    return w;
}
template <uint32_t TYPE>
__device__ __forceinline__ void i8_unpack(uint4 w, float *v) {
    if constexpr (TYPE == SGEMM_I8_FP32) {
        v[0] = __uint_as_float(w.x); v[1] = __uint_as_float(w.y); v[2] = __uint_as_float(w.z); v[3] = __uint_as_float(w.w);
    } else {
        i8_unpack2<TYPE>(w.x, v[0], v[1]);
        i8_unpack2<TYPE>(w.y, v[2], v[3]);
        i8_unpack2<TYPE>(w.z, v[4], v[5]);
        i8_unpack2<TYPE>(w.w, v[6], v[7]);
    }
}
template <uint32_t TYPE>
__device__ __forceinline__ uint4 i8_pack(const float *v) {
    if constexpr (TYPE == SGEMM_I8_FP32)
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    else
        return make_uint4(i8_pack2<TYPE>(v[0], v[1]), i8_pack2<TYPE>(v[2], v[3]), i8_pack2<TYPE>(v[4], v[5]), i8_pack2<TYPE>(v[6], v[7]));
}
// A vector at a row's end (or beginning): the elements of [0, k) only.  One or two of a row's vectors; a loop, to stay out of the way.
template <uint32_t TYPE>
__device__ __forceinline__ uint4 i8_partial_vector(const void *row, int32_t e, int32_t k) {
    constexpr int VE = TYPE == SGEMM_I8_FP32 ? 4 : 8;
    uint64_t w0 = 0, w1 = 0;
#pragma unroll 1
    for (int j = 0; j < VE; ++j) {
        if (e + j < 0 || e + j >= k) continue;
        uint64_t bits;
        if (TYPE == SGEMM_I8_FP32) bits = static_cast<const uint32_t *>(row)[e + j];
        else bits = static_cast<const uint16_t *>(row)[e + j];
        const int shift = j % (VE / 2) * (TYPE == SGEMM_I8_FP32 ? 32 : 16);
        if (j < VE / 2) w0 |= bits << shift;
        else w1 |= bits << shift;
    }
    return make_uint4((uint32_t)w0, (uint32_t)(w0 >> 32), (uint32_t)w1, (uint32_t)(w1 >> 32));
}
template <uint32_t TYPE>
__device__ __forceinline__ void i8_store_partial(void *row, int32_t e, int32_t k, uint4 w) {
    constexpr int VE = TYPE == SGEMM_I8_FP32 ? 4 : 8;
    const uint64_t w0 = w.x | (uint64_t)w.y << 32, w1 = w.z | (uint64_t)w.w << 32;
#pragma unroll 1
    for (int j = 0; j < VE; ++j) {
        if (e + j < 0 || e + j >= k) continue;
        const uint64_t bits = (j < VE / 2 ? w0 : w1) >> (j % (VE / 2) * (TYPE == SGEMM_I8_FP32 ? 32 : 16));
        if (TYPE == SGEMM_I8_FP32) static_cast<uint32_t *>(row)[e + j] = (uint32_t)bits;
        else static_cast<uint16_t *>(row)[e + j] = (uint16_t)bits;
    }
}

// A word of four int8 in which those next to a tie (by `fixed`, see below) are replaced by round(127 p / P), halves to even, in FP64.
// Out of line and four at a time: it is needed for one word in 2000, and the rounding loops stay short.
__device__ __noinline__ uint32_t i8_settle_ties(float v0, float v1, float v2, float v3, uint32_t word, float inverse, float peak, bool all) {
#pragma unroll 1
    for (int j = 0; j < 4; ++j) {
        const float v = j == 0 ? v0 : j == 1 ? v1 : j == 2 ? v2 : v3;
        const uint32_t fixed = 2u * __float_as_uint(fmaf(v, inverse, 384.0f)) + (0x8000u + 4u);
        if ((fixed & 0xFFFFu) <= 8u || all) {
            const uint32_t byte = (uint32_t)(int)rint(127.0 * (double)v / (double)peak) & 0xFFu;
            word = (word & ~(0xFFu << (8 * j))) | (byte << (8 * j));
        }
    }
    return word;
}

// What a thread rounds its elements with: the same for a whole row.
struct I8Rounding {
    float peak, inverse;
    bool pow2, bad, tiny, special;   // special: bad or tiny
    // Four elements to a word of int8
    __device__ __forceinline__ uint32_t word(float v0, float v1, float v2, float v3) const {
        const float v[4] = {v0, v1, v2, v3};
        uint32_t b[4];
        if (pow2) {   // exact: the integer appears in the low mantissa byte
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = __float_as_uint(fmaf(v[j], inverse, I8_ROUND_MAGIC));
            const uint32_t w = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
            return special ? 0u : w;
        }
        // 384 + t has the 15 fraction bits and the 8 integer bits of t side by side in the mantissa; doubled and with 1/2 + 2^-14
        // added they are the upper byte of the low 24 bits, t rounded + 128, and a 16-bit fraction that is at most 8 next to a tie
        uint32_t nearest = 0xFFFFFFFFu;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            b[j] = 2u * __float_as_uint(fmaf(v[j], inverse, 384.0f)) + (0x8000u + 4u);
            nearest = __vminu2(nearest, b[j]);
        }
        uint32_t w = __byte_perm(__byte_perm(b[0], b[1], 0x0062), __byte_perm(b[2], b[3], 0x0062), 0x5410) ^ 0x80808080u;
        if ((nearest & 0xFFFFu) <= 8u || special) w = bad ? 0u : i8_settle_ties(v0, v1, v2, v3, w, inverse, peak, tiny);
        return w;
    }
};

// Scale and rounding of a row from its peak (as FP32 bits).
__device__ __forceinline__ I8Rounding i8_rounding(uint32_t peak_bits, bool pow2, float &scale) {
    I8Rounding r;
    r.peak = __uint_as_float(peak_bits);
    r.pow2 = pow2;
    r.bad = peak_bits > I8_LARGEST_BITS;
    r.tiny = !pow2 && r.peak < I8_TINY && peak_bits != 0u;
    if (pow2) {
        // P = m 2^e: 127 * 2^(e-6) holds it up to m = 127/64, else 2^(e-5); subnormal scales are avoided
        const int e = max((int)(peak_bits >> 23) - 127 - ((peak_bits & 0x7FFFFFu) <= 0x7E0000u ? 6 : 5), -126);
        scale = __uint_as_float((uint32_t)(e + 127) << 23);
        r.inverse = __uint_as_float((uint32_t)(127 - e) << 23);
    } else {
        scale = __fdiv_rn(r.peak, 127.0f);
        r.inverse = r.tiny ? 0.0f : __fdiv_rn(127.0f, r.peak);
    }
    if (peak_bits == 0u) scale = r.inverse = 0.0f;
    if (r.bad) {
        scale = __uint_as_float(0x7FFFFFFFu);
        r.inverse = 0.0f;
        r.tiny = false;
    }
    r.special = r.bad || r.tiny;
    return r;
}

// The norm's scale outside of the ordinary range (out of line: a row in thousands, and its 64-bit code would lie in everybody's way).  The root
// comes from the sum that is in range, P / 127, which has few bits left below the normal numbers, is formed from P * 2^100, and the
// powers of two come off in 64 bits, where nothing on the way can leave the range.
__device__ __noinline__ float i8_norm_scale_far(float peak, float plain, float down, float up, uint32_t k, float inv_k, float eps) {
    if (peak == 0.0f) return 0.0f;
    const float mean = fmaf(plain, inv_k, eps);
    float root;
    double factor = 1.0;
    if (eps < I8_FAINT && plain < I8_FAINT) {
        const float n = (float)k;   // (1 / K could make the mean vanish again)
        root = rsqrtf(fmaf(eps * I8_UP * I8_UP, n, up)) * sqrtf(n);
        factor = (double)I8_UP;
    } else if (!(mean < INFINITY)) {
        root = rsqrtf(fmaf(down, inv_k, eps * I8_DOWN * I8_DOWN));
        factor = (double)I8_DOWN;
    } else {
        root = rsqrtf(mean);
    }
    const bool tiny = peak < I8_TINY;
    const float base = __fdiv_rn(tiny ? peak * 0x1p100f : peak, 127.0f);
    return (float)((double)base * (double)root * (tiny ? factor * 0x1p-100 : factor));
}
// The norm's scale, `base` = P / 127 (NaN where P is out of range) times rsqrt(mean + eps), 0 for a row whose P is 0: the product with 1 / K is off
// by 2^-23 and rsqrtf by 2 of its last places.
template <uint32_t TYPE>
__device__ __forceinline__ float i8_norm_scale(float peak, float base, const float (&sums)[3], uint32_t k, float inv_k, float eps) {
    const float mean = fmaf(sums[0], inv_k, eps);
    if (TYPE == SGEMM_I8_FP16) return peak == 0.0f ? 0.0f : base * rsqrtf(mean);   // squares and products are at least 2^-48, sums stay in range
    if (isnan(base) || (peak >= I8_TINY && mean < INFINITY && (eps >= I8_FAINT || sums[0] >= I8_FAINT))) return base * rsqrtf(mean);
    return i8_norm_scale_far(peak, sums[0], sums[1], sums[2], k, inv_k, eps);
}

// The row's peak over its `tpr` threads (and its first `count` sums, at most SUMS, in a fixed order).
template <int SUMS>
__device__ __forceinline__ void i8_row_reduce(uint32_t &peak_bits, float (&sums)[3], int count, uint32_t tpr) {
    __shared__ float red_sum[3][32];
    __shared__ uint32_t red_max[32];
    peak_bits = __reduce_max_sync(0xffffffffu, peak_bits);
#pragma unroll
    for (int i = 0; i < SUMS; ++i) {
        if (i >= count) break;
#pragma unroll
        for (int d = 16; d; d >>= 1) sums[i] += __shfl_xor_sync(0xffffffffu, sums[i], d);
    }
    if (tpr <= 32) return;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = tpr >> 5, first = warp & ~(warps - 1);
    if (lane == 0) {
        red_max[warp] = peak_bits;
#pragma unroll
        for (int i = 0; i < SUMS; ++i) red_sum[i][warp] = sums[i];
    }
    __syncthreads();
    const bool mine = lane < warps;
    peak_bits = __reduce_max_sync(0xffffffffu, mine ? red_max[first + lane] : 0u);
#pragma unroll
    for (int i = 0; i < SUMS; ++i) {
        if (i >= count) break;
        sums[i] = mine ? red_sum[i][first + lane] : 0.0f;
#pragma unroll
        for (int d = 16; d; d >>= 1) sums[i] += __shfl_xor_sync(0xffffffffu, sums[i], d);
    }
}

// ---- rows in vectors of 16 bytes: a thread takes the t-th of every tpr vectors.  SHIFTED: the row starts `off` elements into its
// first aligned vector (an odd leading dimension, a base inside a larger matrix); the residual and the sum start alike.  Element j of
// vector v is then element v * VE - off + j of the row, and q's aligned words are put together from two lanes' bytes.
template <uint32_t TYPE, int PER, bool NORM, bool SHIFTED>
__device__ __forceinline__ void i8_rows_vector(const I8RowArgs &a) {
    using E = I8Elem<TYPE>;
    using T = typename E::type;
    constexpr int VE = 16 / (int)sizeof(T), NV = PER / VE;
    sgemm_launch_dependents();
    sgemm_grid_dependency_wait();
    const uint32_t row = blockIdx.x * (blockDim.x >> a.tpr_log2) + (threadIdx.x >> a.tpr_log2), t = threadIdx.x & (a.tpr - 1);
    const bool live = row < a.rows;
    const uint64_t r64 = live ? row : 0u;
    const T *x = static_cast<const T *>(a.x) + r64 * a.ldx;
    const int32_t off = SHIFTED ? (int32_t)(((uintptr_t)x & 15u) / sizeof(T)) : 0;
    const T *res = NORM && a.r ? static_cast<const T *>(a.r) + r64 * a.ldr : nullptr;
    const T *g = static_cast<const T *>(a.g);
    T *sum = NORM && a.sum ? static_cast<T *>(a.sum) + r64 * a.lds : nullptr;
    int8_t *q = a.q + r64 * a.ldq;
    const int32_t k = live ? (int32_t)a.k : 0;
    const uint32_t span = a.tpr * PER;
    const uint32_t passes = a.passes;

    // first element of the thread's i-th vector (negative before the row), and whether the vector lies inside the row
    auto first = [&](uint32_t pass, int i) -> int32_t { return (int32_t)(pass * span + (i * a.tpr + t) * VE) - off; };
    auto inside = [&](int32_t e) -> bool { return (!SHIFTED || e >= 0) && e + VE <= k; };
    auto has = [&](int32_t e) -> bool { return (!SHIFTED || e >= 0) && e < k; };
    // 16 bytes of a row, zeros outside of it
    auto load = [&](const T *src, int32_t e, bool whole) -> uint4 {
        if (whole) return *reinterpret_cast<const uint4 *>(src + e);
        return i8_partial_vector<TYPE>(src, e, k);
    };
    uint4 raw[NV];
    float p[NORM ? PER : 1];
    float sums[3] = {0.0f, 0.0f, 0.0f};    // of h^2, of (h * 2^-96)^2 for rows whose squares leave FP32, of (h * 2^92)^2 for those whose squares vanish
    const bool faint = NORM && TYPE != SGEMM_I8_FP16 && a.eps < I8_FAINT;   // the third is taken
    uint32_t peak_pair = 0u;
    float peak = 0.0f;
    auto fetch = [&](uint32_t pass, bool store_sum) {
#pragma unroll
        for (int i = 0; i < NV; ++i) raw[i] = load(x, first(pass, i), inside(first(pass, i)));
        if constexpr (NORM) {
            if (res) {
                uint4 rr[NV];
#pragma unroll
                for (int i = 0; i < NV; ++i) rr[i] = load(res, first(pass, i), inside(first(pass, i)));
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    i8_unpack<TYPE>(raw[i], p + i * VE);
                    float w[VE];
                    i8_unpack<TYPE>(rr[i], w);
#pragma unroll
                    for (int j = 0; j < VE; ++j) p[i * VE + j] = __fadd_rn(p[i * VE + j], w[j]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < NV; ++i) i8_unpack<TYPE>(raw[i], p + i * VE);
            }
            float squares = 0.0f;
#pragma unroll
            for (int j = 0; j < PER; ++j) squares = fmaf(p[j], p[j], squares);
            float small = squares * I8_DOWN * I8_DOWN;
            if (TYPE != SGEMM_I8_FP16 && !(squares < INFINITY)) {   // (squares of FP16 sums cannot leave FP32)
                small = 0.0f;
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    const float v = p[j] * I8_DOWN;
                    small = fmaf(v, v, small);
                }
            }
            sums[0] += squares;
            sums[1] += small;
            if (faint) {
                float large = 0.0f;
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    const float v = p[j] * I8_UP;
                    large = fmaf(v, v, large);
                }
                sums[2] += large;
            }
            if (sum && store_sum) {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int32_t e = first(pass, i);
                    const uint4 w = i8_pack<TYPE>(p + i * VE);
                    if (inside(e)) *reinterpret_cast<uint4 *>(sum + e) = w;
                    else i8_store_partial<TYPE>(sum, e, k, w);
                }
            }
            // gamma comes last, from a cache: its registers are those x and the residual no longer need
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int32_t e = first(pass, i);
                float w[VE];
                if (SHIFTED) {
#pragma unroll
                    for (int j = 0; j < VE; ++j) w[j] = has(e + j) ? E::get(__ldg(g + e + j)) : 0.0f;
                } else {
                    i8_unpack<TYPE>(inside(e) ? __ldg(reinterpret_cast<const uint4 *>(g + e)) : i8_partial_vector<TYPE>(g, e, k), w);
                }
#pragma unroll
                for (int j = 0; j < VE; ++j) {
                    p[i * VE + j] = __fmul_rn(p[i * VE + j], w[j]);
                    peak = i8_max_nan(peak, fabsf(p[i * VE + j]));
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (TYPE == SGEMM_I8_FP32) peak = i8_max_nan(peak, fabsf(__uint_as_float(w[j])));
                    else peak_pair = __vmaxu2(peak_pair, w[j] & 0x7FFF7FFFu);   // as integers NaN > infinity > finite
                }
            }
        }
    };
    fetch(0, passes == 1);
    for (uint32_t pass = 1; pass < passes; ++pass) fetch(pass, false);
    if (!NORM && TYPE != SGEMM_I8_FP32) {
        const uint32_t half = max(peak_pair & 0xFFFFu, peak_pair >> 16);
        float both[2];
        i8_unpack2<TYPE>(half, both[0], both[1]);
        peak = both[0];
    }
    uint32_t peak_bits = i8_abs_bits(peak);
    i8_row_reduce<NORM ? (TYPE == SGEMM_I8_FP16 ? 1 : 3) : 0>(peak_bits, sums, faint ? 3 : 2, a.tpr);
    if (!live) return;   // (a warp has one row: tpr is at least 32)
    float scale;
    const I8Rounding rounding = i8_rounding(peak_bits, !NORM && a.pow2 != 0u, scale);
    if (t == 0) a.scale[row] = NORM ? i8_norm_scale<TYPE>(rounding.peak, scale, sums, a.k, a.inv_k, a.eps) : scale;

    for (uint32_t pass = 0; pass < passes; ++pass) {
        if (passes > 1) fetch(pass, true);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int32_t e = first(pass, i);
            float v[VE];
            if constexpr (NORM) {
#pragma unroll
                for (int j = 0; j < VE; ++j) v[j] = p[i * VE + j];
            } else {
                i8_unpack<TYPE>(raw[i], v);
            }
            uint32_t word[VE / 4];
#pragma unroll
            for (int w = 0; w < VE / 4; ++w) word[w] = rounding.word(v[4 * w], v[4 * w + 1], v[4 * w + 2], v[4 * w + 3]);
            if constexpr (!SHIFTED) {
                if (inside(e)) {
                    if constexpr (VE == 8) *reinterpret_cast<uint2 *>(q + e) = make_uint2(word[0], word[1]);
                    else *reinterpret_cast<uint32_t *>(q + e) = word[0];
                } else {
#pragma unroll
                    for (int j = 0; j < VE; ++j)
                        if (has(e + j)) q[e + j] = (int8_t)(word[j / 4] >> (8 * (j & 3)));
                }
            } else {
                // the aligned word of q that holds this vector's first byte: its first d bytes are the previous lane's last ones
                const uint32_t lane = threadIdx.x & 31u, d = (uint32_t)((uintptr_t)(q + e) & (VE - 1));
                uint64_t mine, before;
                if constexpr (VE == 8) {
                    mine = ((uint64_t)word[1] << 32) | word[0];
                    before = __shfl_up_sync(0xffffffffu, mine, 1);
                } else {
                    mine = word[0];
                    before = __shfl_up_sync(0xffffffffu, word[0], 1);
                }
                const bool whole = e - (int32_t)d >= 0 && e - (int32_t)d + VE <= k && (lane != 0u || d == 0u);
                if (whole) {
                    const uint64_t joined = d ? (mine << (8 * d)) | (before >> (8 * (VE - d))) : mine;
                    if constexpr (VE == 8) *reinterpret_cast<uint64_t *>(q + e - d) = joined;
                    else *reinterpret_cast<uint32_t *>(q + e - d) = (uint32_t)joined;
                }
                // bytes that no whole word took: those of this lane's word where it is not whole, and the last d of a vector whose next lane
                // is in another warp or has no whole word
                const bool next_whole = lane != 31u && e + VE - (int32_t)d >= 0 && e + 2 * VE - (int32_t)d <= k;
#pragma unroll
                for (int j = 0; j < VE; ++j) {
                    const bool own = j < (int)(VE - d);   // in the word of this lane, else in the next one's
                    if (!(own ? whole : next_whole) && has(e + j)) q[e + j] = (int8_t)(mine >> (8 * j));
                }
            }
        }
    }
}

// ---- rows that start anywhere: a thread's elements are the t-th of every tpr, so that a warp's loads and stores are
// consecutive elements
template <uint32_t TYPE, bool NORM>
__device__ __forceinline__ void i8_rows_scalar(const I8RowArgs &a) {
    using E = I8Elem<TYPE>;
    using T = typename E::type;
    constexpr int PER = 32;
    sgemm_launch_dependents();
    sgemm_grid_dependency_wait();
    const uint32_t row = blockIdx.x * (blockDim.x >> a.tpr_log2) + (threadIdx.x >> a.tpr_log2), t = threadIdx.x & (a.tpr - 1);
    const bool live = row < a.rows;
    const uint64_t r64 = live ? row : 0u;
    const T *x = static_cast<const T *>(a.x) + r64 * a.ldx;
    const T *res = NORM && a.r ? static_cast<const T *>(a.r) + r64 * a.ldr : nullptr;
    const T *g = static_cast<const T *>(a.g);
    T *sum = NORM && a.sum ? static_cast<T *>(a.sum) + r64 * a.lds : nullptr;
    int8_t *q = a.q + r64 * a.ldq;
    const uint32_t k = live ? a.k : 0u, span = a.tpr * PER;
    const uint32_t passes = a.passes;
    float p[PER];
    float sums[3] = {0.0f, 0.0f, 0.0f};
    const bool faint = NORM && TYPE != SGEMM_I8_FP16 && a.eps < I8_FAINT;
    uint32_t peak_bits = 0u;
    auto fetch = [&](uint32_t pass, bool store_sum) {
        const uint32_t first = pass * span + t;
#pragma unroll
        for (int j = 0; j < PER; ++j) p[j] = first + j * a.tpr < k ? E::get(x[first + j * a.tpr]) : 0.0f;
        if constexpr (NORM) {
            if (res) {
                float r[PER];
#pragma unroll
                for (int j = 0; j < PER; ++j) r[j] = first + j * a.tpr < k ? E::get(res[first + j * a.tpr]) : 0.0f;
#pragma unroll
                for (int j = 0; j < PER; ++j) p[j] = __fadd_rn(p[j], r[j]);
            }
            if (sum && store_sum) {
#pragma unroll
                for (int j = 0; j < PER; ++j)
                    if (first + j * a.tpr < k) sum[first + j * a.tpr] = E::put(p[j]);
            }
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                sums[0] = fmaf(p[j], p[j], sums[0]);
                if (TYPE != SGEMM_I8_FP16) {
                    const float small = p[j] * I8_DOWN;
                    sums[1] = fmaf(small, small, sums[1]);
                    if (faint) {
                        const float large = p[j] * I8_UP;
                        sums[2] = fmaf(large, large, sums[2]);
                    }
                }
                p[j] = __fmul_rn(p[j], first + j * a.tpr < k ? E::get(__ldg(g + first + j * a.tpr)) : 0.0f);
            }
        }
    };
    for (uint32_t pass = 0; pass < passes; ++pass) {
        fetch(pass, passes == 1);
#pragma unroll
        for (int j = 0; j < PER; ++j) peak_bits = max(peak_bits, i8_abs_bits(p[j]));
    }
    i8_row_reduce<NORM ? (TYPE == SGEMM_I8_FP16 ? 1 : 3) : 0>(peak_bits, sums, faint ? 3 : 2, a.tpr);
    if (!live) return;
    float scale;
    const I8Rounding rounding = i8_rounding(peak_bits, !NORM && a.pow2 != 0u, scale);
    if (t == 0) a.scale[row] = NORM ? i8_norm_scale<TYPE>(rounding.peak, scale, sums, a.k, a.inv_k, a.eps) : scale;
    for (uint32_t pass = 0; pass < passes; ++pass) {
        if (passes > 1) fetch(pass, true);
        const uint32_t first = pass * span + t;
#pragma unroll
        for (int w = 0; w < PER / 4; ++w) {
            const uint32_t word = rounding.word(p[4 * w], p[4 * w + 1], p[4 * w + 2], p[4 * w + 3]);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (first + (4 * w + j) * a.tpr < k) q[first + (4 * w + j) * a.tpr] = (int8_t)(word >> (8 * j));
        }
    }
}

// One kernel per element type and elements per thread; the host picks by K, alignment and row count.
#define I8_ROW_KERNEL(NAME, THREADS, BLOCKS, BODY, ...)                                                                            \
    extern "C" __global__ void __launch_bounds__(THREADS, BLOCKS) NAME(const __grid_constant__ I8RowArgs a) { BODY<__VA_ARGS__>(a); }
// (blocks: how many of 32 elements a thread an SM is to hold, which sets the registers a thread gets)
#define I8_ROW_KERNELS(OP, NORM, NAME, TYPE, BLOCKS)                                      \
    I8_ROW_KERNEL(OP##_##NAME##_v1, 1024, 1, i8_rows_vector, TYPE, 8, NORM, false)        \
    I8_ROW_KERNEL(OP##_##NAME##_v2, 512, 2, i8_rows_vector, TYPE, 16, NORM, false)        \
    I8_ROW_KERNEL(OP##_##NAME##_v4, 256, BLOCKS, i8_rows_vector, TYPE, 32, NORM, false)        \
    I8_ROW_KERNEL(OP##_##NAME##_u4, 256, BLOCKS, i8_rows_vector, TYPE, 32, NORM, true)         \
    I8_ROW_KERNEL(OP##_##NAME##_s4, 256, 2, i8_rows_scalar, TYPE, NORM)
I8_ROW_KERNELS(i8_quantize, false, fp32, SGEMM_I8_FP32, 3)
I8_ROW_KERNELS(i8_quantize, false, fp16, SGEMM_I8_FP16, 4)
I8_ROW_KERNELS(i8_quantize, false, bf16, SGEMM_I8_BF16, 4)
I8_ROW_KERNELS(i8_rmsnorm, true, fp32, SGEMM_I8_FP32, 2)
I8_ROW_KERNELS(i8_rmsnorm, true, fp16, SGEMM_I8_FP16, 4)
I8_ROW_KERNELS(i8_rmsnorm, true, bf16, SGEMM_I8_BF16, 4)

// ---------------------------------------------------------------------------------------------
// restore: every thread widens 16 consecutive int8 of a row (aligned q and output), or, for rows that start anywhere, the int8
// of one aligned 16-byte vector of the output, put together from the aligned words of q that hold them.
// ---------------------------------------------------------------------------------------------
template <uint32_t TYPE>
__device__ __forceinline__ void i8_restore_vector(const int8_t *q, const float *scale, void *out, uint32_t k, uint32_t rows,
                                                  uint32_t ldq, uint32_t ldo) {
    using E = I8Elem<TYPE>;
    using T = typename E::type;
    sgemm_launch_dependents();
    sgemm_grid_dependency_wait();
    const uint32_t units = (k + 15) / 16;   // of a row
    const uint64_t total = (uint64_t)units * rows, stride = (uint64_t)gridDim.x * blockDim.x;
    for (uint64_t at = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; at < total; at += stride) {
        const uint32_t row = total <= 0xFFFFFFFFull ? (uint32_t)at / units : (uint32_t)(at / units);
        const uint32_t e = (uint32_t)(at - (uint64_t)row * units) * 16;
        const float s = scale[row];
        const int8_t *src = q + (uint64_t)row * ldq + e;
        T *dst = static_cast<T *>(out) + (uint64_t)row * ldo + e;
        if (e + 16 <= k) {
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
            for (uint32_t j = 0; e + j < k; ++j) dst[j] = E::put((float)src[j] * s);
        }
    }
}
template <uint32_t TYPE>
__device__ __forceinline__ void i8_restore_shifted(const int8_t *q, const float *scale, void *out, uint32_t k, uint32_t rows,
                                                   uint32_t ldq, uint32_t ldo) {
    using E = I8Elem<TYPE>;
    using T = typename E::type;
    constexpr int VE = 16 / (int)sizeof(T);
    sgemm_launch_dependents();
    sgemm_grid_dependency_wait();
    const uint32_t units = (k + VE - 1) / VE + 1;   // aligned vectors a row of any offset may touch
    const uint64_t total = (uint64_t)units * rows, stride = (uint64_t)gridDim.x * blockDim.x;
    for (uint64_t at = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; at < total; at += stride) {
        const uint32_t row = total <= 0xFFFFFFFFull ? (uint32_t)at / units : (uint32_t)(at / units);
        T *dst = static_cast<T *>(out) + (uint64_t)row * ldo;
        const int8_t *src = q + (uint64_t)row * ldq;
        const int64_t e = (int64_t)(at - (uint64_t)row * units) * VE - (int64_t)(((uintptr_t)dst & 15u) / sizeof(T));
        const float s = scale[row];
        const uint32_t c = (uint32_t)((uintptr_t)(src + e) & 3u);   // bytes of the first word before the vector
        if (e - (int64_t)c >= 0 && e + VE + 4 <= (int64_t)k) {
            const uint32_t *w = reinterpret_cast<const uint32_t *>(src + e - c);
            uint32_t in[VE / 4 + 1];
#pragma unroll
            for (int i = 0; i <= VE / 4; ++i) in[i] = w[i];
            uint4 o;
            T *po = reinterpret_cast<T *>(&o);
#pragma unroll
            for (int i = 0; i < VE / 4; ++i) {
                float v[4];
                i8_widen4(__funnelshift_r(in[i], in[i + 1], 8 * c), v);
#pragma unroll
                for (int j = 0; j < 4; ++j) po[4 * i + j] = E::put(v[j] * s);
            }
            *reinterpret_cast<uint4 *>(dst + e) = o;
        } else {
            for (int j = 0; j < VE; ++j)
                if (e + j >= 0 && e + j < (int64_t)k) dst[e + j] = E::put((float)src[e + j] * s);
        }
    }
}
#define I8_RESTORE_KERNEL(NAME, BODY, TYPE)                                                                            \
    extern "C" __global__ void __launch_bounds__(256) NAME(const int8_t *q, const float *scale, void *out, uint32_t k, \
                                                           uint32_t rows, uint32_t ldq, uint32_t ldo) {                \
        BODY<TYPE>(q, scale, out, k, rows, ldq, ldo);                                                                  \
    }
I8_RESTORE_KERNEL(i8_restore_fp32_v, i8_restore_vector, SGEMM_I8_FP32)
I8_RESTORE_KERNEL(i8_restore_fp16_v, i8_restore_vector, SGEMM_I8_FP16)
I8_RESTORE_KERNEL(i8_restore_bf16_v, i8_restore_vector, SGEMM_I8_BF16)
I8_RESTORE_KERNEL(i8_restore_fp32_u, i8_restore_shifted, SGEMM_I8_FP32)
I8_RESTORE_KERNEL(i8_restore_fp16_u, i8_restore_shifted, SGEMM_I8_FP16)
I8_RESTORE_KERNEL(i8_restore_bf16_u, i8_restore_shifted, SGEMM_I8_BF16)
