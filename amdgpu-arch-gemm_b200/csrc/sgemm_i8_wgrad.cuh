// ---------------------------------------------------------------------------------------------
// Weight gradient from an activation checkpoint in 8 bits (tcgen05 kind::f16, FP32 accumulators in TMEM).
//
//   D[i, j] = alpha * sum_t V(q[i, t], s[t]) * G[j, t] + beta * C[i, j]         i < M features, j < N channels, t < T tokens
//
// q is M x T int8 with one scale per token (column), G is N x T in FP16 or BF16, both column-major: features and channels are
// contiguous, tokens are the contraction.  C and D are M x N column-major, so a channel's features are contiguous.
// V(q, s) is s * q rounded to G's type, the value i8_restore gives.  With power-of-two scales it is s * q itself (7
// significant bits), and the only rounding besides the FP32 sum is the last one, to D's type.  The 16-bit copy of the
// activations exists in shared memory only: the checkpoint is read as 8 bits.
//
// Roles, as in the in-kernel split of the FP32 kernel: a TMA producer brings a stage of I8W_BK tokens (raw int8 tile, G tile), a
// second warp their scales (4-byte asynchronous copies: any base, and no trip to memory inside the widening warps); two groups of
// eight warps, taking stages in turn, widen the raw tile into an A operand; one thread of the pair's leader issues the MMAs;
// eight warps drain the accumulators.  CTA pairs (cta_group::2) work on 256 features x 256 channels: each CTA widens 128
// features and stages 128 channels, so a widened element meets 256 channels.
//
// What bounds it: 4096 x 4096 over 8192 tokens takes 236 us (1.16 PFLOP/s; the same kernel without the widening's work 191).  A stage's
// MMAs need 512 cycles, its traffic through shared memory (operands 32 KB, TMA 24 KB, widening 24 KB) 640 at 128 bytes a cycle, and the
// widening warps' chains of dependent instructions add their latency.  The warps that wait cost little (naps between their
// looks at a barrier changed nothing), and so does the depth of the rings (5 widened tiles and 5 stages: 242 us).
//
// Both operands are MN-major 16-bit tiles (a row of 128 bytes = 64 features or channels of one token, 128-byte swizzle,
// repeating unit 8 tokens: SBO = 1024; chunks of 64 features I8W_BK * 128 bytes apart: LBO); one MMA takes 16 tokens = 2048 bytes.
//
// The tensor core adds to its accumulator with truncation, so a long sum drifts toward zero: every I8W_CHAIN stages (32 additions) the
// issuer turns to the other TMEM buffer and the epilogue warps add the finished chain to a running sum in registers, rounding to
// nearest, in a fixed order.
//
// Few tiles and many tokens: S = 2, 3 or 4 pairs of a cluster take S parts of the tokens of one tile.  Each leaves its sums in
// its shared memory and after a cluster barrier adds up its share of the columns over all parts, in the order of the
// parts: no workspace, no atomics, the same bits every time.
// ---------------------------------------------------------------------------------------------
struct I8WgradArgs {
    const int8_t *q;
    const float *scale;
    const void *g;
    const void *c;
    void *d;
    uint32_t *status;
    uint32_t m, n, tokens, ldq, ldg, ldc, ldd;
    uint32_t g_type, d_type;
    float alpha, beta;
    uint32_t tiles_m, tiles_n;
};

#define I8W_RAW_BYTES (128 * I8W_BK)
#define I8W_OP_BYTES (2 * 128 * I8W_BK)            // a widened tile, or G's
#define I8W_CHUNK_BYTES (I8W_BK * 128)             // 64 features (channels) of a tile
#define I8W_REGS_SMALL 40
#define I8W_REGS_WIDEN 40
#define I8W_REGS_EPI 152
static_assert(I8W_REGS_SMALL + 4 * I8W_REGS_WIDEN + 2 * I8W_REGS_EPI <= 7 * I8W_LAUNCH_REGS,
              "the register hand-over must not ask for more than the launch allocated");
static_assert(I8W_THREADS == 896 && I8W_SMEM <= 232448, "seven groups of four warps, one CTA per SM");
static_assert(I8W_RING_BYTES >= 128 * 256 * 4, "a part's sums must fit the drained rings");
// shared memory: widened A tiles, then G tiles, raw tiles and scales of the stages in flight
#define I8W_G_OFFSET (I8W_A_STAGES * I8W_OP_BYTES)
#define I8W_RAW_OFFSET (I8W_G_OFFSET + I8W_STAGES * I8W_OP_BYTES)
#define I8W_SCALE_OFFSET (I8W_RAW_OFFSET + I8W_STAGES * I8W_RAW_BYTES)
static_assert(I8W_SCALE_OFFSET + I8W_STAGES * 4 * I8W_BK == I8W_RING_BYTES, "the rings as the host sizes them");

// kind::f16 instruction descriptor: FP32 accumulator, A and B of one 16-bit type (0 = FP16, 1 = BF16), both MN-major, 256 x 256
__device__ __forceinline__ uint32_t i8w_idesc(uint32_t g_type) {
    const uint32_t fmt = g_type == SGEMM_I8_BF16 ? 1u : 0u;
    return (1u << 4) | (fmt << 7) | (fmt << 10) | (1u << 15) | (1u << 16) | ((256u >> 3) << 17) | ((256u >> 4) << 24);
}

// two values to one word of G's type, round to nearest even
__device__ __forceinline__ uint32_t i8w_pack(float lo, float hi, uint32_t g_type) {
    uint32_t w;
    if (g_type == SGEMM_I8_BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    return w;
}

// Widening of the four int8 of a word.  The order within a group of four features is 0, 2, 1, 3 (bytes 0 and 2 of a word lie where the
// two halves of a packed 16-bit pair want them, bytes 1 and 3 after one shift); it is a permutation of the rows of the MMA's A operand,
// undone where the epilogue maps lanes to features (i8w_feature).
//
// Power-of-two scales (what checkpoints have; 0 too) go in packed 16-bit arithmetic, exactly:
//   BF16: 7 bits of q under the exponent of 2^7 give 128 + (q mod 128); adding -128, or -256 where q is negative (its sign bit
//         is the lowest exponent bit of that constant), leaves q, and the product with s is exact.
//   FP16: q + 128 under the exponent of 2^10 gives 1152 + q; one fused multiply-add with s and -1152 s gives s * q, rounded once
//         (subnormal results), as long as 1152 s is in range and s itself is a number of the type.
// 2.25 and 1.25 instructions an element against 3.75 through FP32, which all other scales take.
// Whether a thread's scales are such for G's type (the product of FP16 leaves 0 and scales outside of 2^-24 .. 2^5 to the general form).
__device__ __forceinline__ bool i8w_plain_scales(const float (&s)[2], uint32_t g_type) {
    uint32_t all = 0u, far = 0u;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        all |= __float_as_uint(s[i]);
        far = max(far, __float_as_uint(s[i]) - 0x33800000u);
    }
    return (all & 0x807FFFFFu) == 0u && (g_type == SGEMM_I8_BF16 || far <= 0x42000000u - 0x33800000u);
}
struct I8WidenBf16 {
    __nv_bfloat162 s2;
    __device__ __forceinline__ explicit I8WidenBf16(float s) {
        const uint32_t w = __byte_perm(__float_as_uint(s), 0u, 0x3232);
        s2 = *reinterpret_cast<const __nv_bfloat162 *>(&w);
    }
    __device__ __forceinline__ uint32_t pair(uint32_t w) const {
        const uint32_t m = (w & 0x007F007Fu) | 0x43004300u, c = (w & 0x00800080u) | 0xC300C300u;
        const __nv_bfloat162 v = __hmul2(__hadd2(*reinterpret_cast<const __nv_bfloat162 *>(&m), *reinterpret_cast<const __nv_bfloat162 *>(&c)), s2);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
    __device__ __forceinline__ uint2 word(uint32_t w) const { return make_uint2(pair(w), pair(w >> 8)); }
};
struct I8WidenFp16 {
    __half2 s2, o2;
    __device__ __forceinline__ explicit I8WidenFp16(float s) : s2(__float2half2_rn(s)), o2(__float2half2_rn(-1152.0f * s)) {}
    __device__ __forceinline__ uint32_t pair(uint32_t m) const {
        const __half2 v = __hfma2(*reinterpret_cast<const __half2 *>(&m), s2, o2);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
    __device__ __forceinline__ uint2 word(uint32_t w) const {
        const uint32_t u = w ^ 0x80808080u;
        return make_uint2(pair(__byte_perm(u, 0x64646464u, 0x4240)), pair(__byte_perm(u, 0x64646464u, 0x4341)));
    }
};
struct I8WidenAny {   // through FP32, one rounding
    float s;
    uint32_t g_type;
    __device__ __forceinline__ uint2 word(uint32_t w) const {
        float v[4];
        i8_widen4(w, v);
        return make_uint2(i8w_pack(v[0] * s, v[2] * s, g_type), i8w_pack(v[1] * s, v[3] * s, g_type));
    }
};
// Feature (row of a 128-row half of the tile) at position `p` of the A operand.
__device__ __forceinline__ uint32_t i8w_feature(uint32_t p) { return (p & ~3u) | ((p & 1u) << 1) | ((p >> 1) & 1u); }

// The running sum of one lane: 128 columns of one row, two to a 64-bit register pair.
__device__ __forceinline__ uint64_t i8w_pair(float lo, float hi) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}
__device__ __forceinline__ float2 i8w_unpair(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
// sum2 += beta * C, eight columns at a time (as many as there are registers for).  L2 is asked for all of them first: lane l of the warp
// covers columns l, l + 32, ... of its 32 rows.
template <uint32_t TYPE>
__device__ __forceinline__ void i8w_add_c(uint64_t (&sum2)[64], const I8WgradArgs &a, uint32_t row, uint32_t row_first, uint32_t col0) {
    using E = I8Elem<TYPE>;
    using T = typename E::type;
    const T *c = static_cast<const T *>(a.c) + (uint64_t)col0 * a.ldc;
    const uint32_t cols = col0 < a.n ? min(128u, a.n - col0) : 0u;
    if (row_first < a.m) {
        const uint32_t row_last = min(row_first + 31u, a.m - 1u);
        for (uint32_t col = threadIdx.x & 31u; col < cols; col += 32) {
            asm volatile("prefetch.global.L2 [%0];" ::"l"(c + row_first + (uint64_t)col * a.ldc));
            asm volatile("prefetch.global.L2 [%0];" ::"l"(c + row_last + (uint64_t)col * a.ldc));
        }
    }
    const uint32_t mine = row < a.m ? cols : 0u;
    c += row;
#pragma unroll
    for (int block = 0; block < 16; ++block) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = block * 8 + e < mine ? E::get(c[(uint64_t)e * a.ldc]) : 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) sum2[block * 4 + e] = i8w_pair(a.beta * v[2 * e], a.beta * v[2 * e + 1]);
        c += (uint64_t)8 * a.ldc;
        asm volatile("" : "+l"(c)::"memory");
    }
}
template <uint32_t TYPE>
__device__ __forceinline__ void i8w_store_sums(const uint64_t (&sum2)[64], const I8WgradArgs &a, uint32_t row, uint32_t col0) {
    using E = I8Elem<TYPE>;
    typename E::type *d = static_cast<typename E::type *>(a.d) + row + (uint64_t)col0 * a.ldd;
    const uint32_t cols = row < a.m && col0 < a.n ? min(128u, a.n - col0) : 0u;
#pragma unroll
    for (int j = 0; j < 64; ++j) {
        const float2 v = i8w_unpair(sum2[j]);
        if (2 * j < cols) *d = E::put(v.x);
        d += a.ldd;
        if (2 * j + 1 < cols) *d = E::put(v.y);
        d += a.ldd;
    }
}

extern "C" __global__ void __launch_bounds__(I8W_THREADS, 1)
i8_wgrad(const __grid_constant__ I8WgradArgs a, const __grid_constant__ I8TensorMap map_q, const __grid_constant__ I8TensorMap map_g) {
    extern __shared__ uint8_t i8w_smem_raw[];
    const uint32_t smem_base = (i8_smem_u32(i8w_smem_raw) + 1023u) & ~1023u;
    uint8_t *generic_base = i8w_smem_raw + (smem_base - i8_smem_u32(i8w_smem_raw));
    // barriers: full[S] and empty[S] of the stages in flight, ready[A] and free[A] of the widened tiles, tmem_full[2], tmem_empty[2]
    const uint32_t bar_full = smem_base + I8W_RING_BYTES, bar_empty = bar_full + 8 * I8W_STAGES;
    const uint32_t bar_ready = bar_empty + 8 * I8W_STAGES, bar_free = bar_ready + 8 * I8W_A_STAGES;
    const uint32_t bar_tfull = bar_free + 8 * I8W_A_STAGES, bar_tempty = bar_tfull + 16;
    constexpr uint32_t kBarrierBytes = 16 * I8W_STAGES + 16 * I8W_A_STAGES + 32;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(generic_base + I8W_RING_BYTES + kBarrierBytes);
    volatile uint32_t *abort_flag = tmem_slot + 1;
    static_assert(kBarrierBytes + 8 <= 256, "barrier block size");
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const I8Wait waiter{abort_flag, a.status, I8_TIMEOUT_NS};
    // the cluster holds S pairs; pair z takes the z-th part of the tokens, its even CTA leads
    const uint32_t cluster_rank = i8_cluster_rank(), parts = i8_cluster_size() / 2, part = cluster_rank / 2, rank = cluster_rank & 1u;
    const uint32_t leader = cluster_rank & ~1u;
    const uint32_t unit0 = blockIdx.x / (2 * parts), unit_stride = gridDim.x / (2 * parts);
    const uint32_t num_tiles = a.tiles_m * a.tiles_n;
    const uint32_t blocks = (a.tokens + I8W_BK - 1) / I8W_BK;
    const uint32_t kb_begin = (uint32_t)((uint64_t)blocks * part / parts), kb_end = (uint32_t)((uint64_t)blocks * (part + 1) / parts);

    if (threadIdx.x == 0) {
        for (int s = 0; s < I8W_STAGES; ++s) {
            i8_mbar_init(bar_full + 8 * s, 1 + 32);   // the TMA producer and the lanes of the scales' warp
            i8_mbar_init(bar_empty + 8 * s, 1);
        }
        for (int s = 0; s < I8W_A_STAGES; ++s) {
            i8_mbar_init(bar_ready + 8 * s, 8 * 2);
            i8_mbar_init(bar_free + 8 * s, 1);
        }
        for (int i = 0; i < 2; ++i) {
            i8_mbar_init(bar_tfull + 8 * i, 1);
            i8_mbar_init(bar_tempty + 8 * i, 8 * 2);
        }
        *abort_flag = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        i8_prefetch_map(&map_q);
        i8_prefetch_map(&map_g);
    }
    if (warp == 1) i8_tmem_alloc<2>(i8_smem_u32(tmem_slot), 512);
    i8_fence_before();
    i8_cluster_sync();
    i8_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    sgemm_launch_dependents();
    sgemm_grid_dependency_wait();

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(I8W_REGS_SMALL));
        if (warp == 0) {
            // ---- TMA producer: each CTA's loads report to its own "full" barrier (it widens what it loaded)
            uint32_t stage = 0, phase = 0;
            bool alive = true;
            for (uint32_t tile = unit0; alive && tile < num_tiles; tile += unit_stride) {
                uint32_t tx, ty;
                sgemm_tile_raster(tile, a.tiles_m, a.tiles_n, OPT_WGM, tx, ty);
                const int32_t m0 = (int32_t)(tx * 256 + rank * 128), n0 = (int32_t)(ty * 256 + rank * 128);
                for (uint32_t kb = kb_begin; kb < kb_end; ++kb) {
                    if (!i8_wait_warp(waiter, bar_empty + 8 * stage, phase ^ 1u, 0x120u + stage, tile, kb)) { alive = false; break; }
                    const uint32_t sg = smem_base + I8W_G_OFFSET + stage * I8W_OP_BYTES, raw = smem_base + I8W_RAW_OFFSET + stage * I8W_RAW_BYTES;
                    const uint32_t full = bar_full + 8 * stage;
                    const int32_t t0 = (int32_t)(kb * I8W_BK);
                    if (i8_elect()) {
                        i8_mbar_expect_tx(full, I8W_RAW_BYTES + I8W_OP_BYTES);
                        i8_tma_load(raw, &map_q, full, m0, t0);
                        i8_tma_load(sg, &map_g, full, n0, t0);
                        i8_tma_load(sg + I8W_CHUNK_BYTES, &map_g, full, n0 + 64, t0);
                    }
                    if (++stage == I8W_STAGES) { stage = 0; phase ^= 1u; }
                }
            }
        } else if (warp == 2) {   // ---- scales: lane l brings those of tokens l and l + 32 of the stage, zeros beyond the last token
            uint32_t stage = 0, phase = 0;
            bool alive = true;
            for (uint32_t tile = unit0; alive && tile < num_tiles; tile += unit_stride) {
                for (uint32_t kb = kb_begin; kb < kb_end; ++kb) {
                    alive = i8_wait_warp(waiter, bar_empty + 8 * stage, phase ^ 1u, 0x620u + stage, tile, kb);
                    if (!alive) break;
                    const uint32_t dst = smem_base + I8W_SCALE_OFFSET + stage * (4 * I8W_BK) + lane * 4;
#pragma unroll
                    for (int i = 0; i < I8W_BK / 32; ++i) {
                        const uint32_t token = kb * I8W_BK + i * 32 + lane;
                        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + i * 128),
                                     "l"(a.scale + min(token, a.tokens - 1u)), "r"(token < a.tokens ? 4u : 0u) : "memory");
                    }
                    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar_full + 8 * stage) : "memory");
                    if (++stage == I8W_STAGES) { stage = 0; phase ^= 1u; }
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        } else if (warp == 1) {
            if (rank == 0) {   // ---- MMA issuer
                const uint32_t idesc = i8w_idesc(a.g_type);
                const uint16_t pair_mask = (uint16_t)(3u << leader);
                const uint64_t desc_a0 = i8_smem_desc(smem_base, I8W_CHUNK_BYTES, 1024), desc_g0 = desc_a0 + I8W_G_OFFSET / 16;
                uint64_t desc_a = desc_a0, desc_g = desc_g0;
                uint32_t stage = 0, widened = 0, phase = 0, handover = 0;   // phase: of the widened tiles
                bool alive = true;
                for (uint32_t tile = unit0; alive && tile < num_tiles; tile += unit_stride) {
                    for (uint32_t kb = kb_begin; alive && kb < kb_end; ++handover) {
                        const uint32_t buf = handover & 1u, acc_phase = (handover >> 1) & 1u;
                        if (!i8_wait_warp(waiter, bar_tempty + 8 * buf, acc_phase ^ 1u, 0x220u + buf, tile, kb)) { alive = false; break; }
                        i8_fence_after();
                        const uint32_t chain_begin = kb, chain_end = min(kb_end, kb + I8W_CHAIN);
                        for (; kb < chain_end; ++kb) {
                            // (a widened tile's "ready" implies that both CTAs' G tiles have landed)
                            if (!i8_wait_warp(waiter, bar_ready + 8 * widened, phase, 0x320u + widened, tile, kb)) { alive = false; break; }
                            i8_fence_after();
                            if (i8_elect()) {
#pragma unroll
                                for (int kk = 0; kk < I8W_BK / 16; ++kk)   // 16 tokens are 2048 bytes of a chunk
                                    i8_mma_f16_pair(tmem_base + buf * 256, desc_a + kk * (2048 / 16), desc_g + kk * (2048 / 16), idesc,
                                                    (kb == chain_begin && kk == 0) ? 0u : 1u);
                                i8_commit<2>(bar_free + 8 * widened, pair_mask);
                                i8_commit<2>(bar_empty + 8 * stage, pair_mask);
                                if (kb + 1 == chain_end) i8_commit<2>(bar_tfull + 8 * buf, pair_mask);
                            }
                            desc_a += I8W_OP_BYTES / 16;
                            desc_g += I8W_OP_BYTES / 16;
                            if (++stage == I8W_STAGES) {
                                stage = 0;
                                desc_g = desc_g0;
                            }
                            if (++widened == I8W_A_STAGES) {
                                widened = 0;
                                phase ^= 1u;
                                desc_a = desc_a0;
                            }
                        }
                    }
                }
            }
        }
    } else if (warp >= 12) {
        // ---- widening: thread t of 256 takes features 16 (t % 8) .. + 15 of tokens t / 8 and t / 8 + 32 (the two chunks of 64
        // features of a token in swapped pairs: the eight lanes of a token pair's row then hit eight different units of the swizzled
        // rows they write).  Four warps per scheduler with two vectors each: with half the warps and twice the vectors 4096 x 4096
        // over 8192 tokens took 262 us instead of 248, with twelve warps away from the MMA issuer's scheduler 249 instead of 236
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(I8W_REGS_WIDEN));
        const uint32_t group = (warp - 12) >> 3, t = (threadIdx.x - 384) & 255u, unit = t & 7u, chunk = unit >> 2, tok = (t >> 3) ^ chunk;
        const uint32_t ready_base = i8_map_to_cta(bar_ready, leader);
        const uint32_t swizzled = (((unit & 3u) * 2) ^ (tok & 7u)) << 4;   // first of the thread's two units; the second is ^ 16
        uint32_t stage = 0, phase = 0, widened = 0, free_phase = 1, turn = 0;
        bool alive = true;
        for (uint32_t tile = unit0; alive && tile < num_tiles; tile += unit_stride) {
            for (uint32_t kb = kb_begin; kb < kb_end; ++kb, ++turn) {
                const uint32_t from = stage, from_phase = phase, to = widened, to_phase = free_phase;
                if (++stage == I8W_STAGES) { stage = 0; phase ^= 1u; }
                if (++widened == I8W_A_STAGES) { widened = 0; free_phase ^= 1u; }
                if ((turn & 1u) != group) continue;
                alive = i8_wait_warp(waiter, bar_free + 8 * to, to_phase, 0x720u + to, tile, kb) &&
                        i8_wait_warp(waiter, bar_full + 8 * from, from_phase, 0x520u + from, tile, kb);
                if (!alive) break;
                const uint32_t raw = smem_base + I8W_RAW_OFFSET + from * I8W_RAW_BYTES + tok * 128 + unit * 16;
                const uint32_t scales = smem_base + I8W_SCALE_OFFSET + from * (4 * I8W_BK) + tok * 4;
                const uint32_t dst = smem_base + to * I8W_OP_BYTES + chunk * I8W_CHUNK_BYTES + tok * 128;
                // (all loads before the first store)
                const uint4 w[2] = {i8_lds4(raw), i8_lds4(raw + 32 * 128)};
                const float s[2] = {i8_ldsf(scales), i8_ldsf(scales + 32 * 4)};
                auto store = [&](int i, const auto &widen) {
                    const uint2 w0 = widen.word(w[i].x), w1 = widen.word(w[i].y);
                    i8_sts4(dst + i * 32 * 128 + swizzled, w0.x, w0.y, w1.x, w1.y);
                    const uint2 w2 = widen.word(w[i].z), w3 = widen.word(w[i].w);
                    i8_sts4(dst + i * 32 * 128 + (swizzled ^ 16u), w2.x, w2.y, w3.x, w3.y);
                };
                if (!i8w_plain_scales(s, a.g_type)) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) store(i, I8WidenAny{s[i], a.g_type});
                } else if (a.g_type == SGEMM_I8_BF16) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) store(i, I8WidenBf16(s[i]));
                } else {
#pragma unroll
                    for (int i = 0; i < 2; ++i) store(i, I8WidenFp16(s[i]));
                }
                // generic-proxy writes -> visible to the tensor core (async proxy), then hand the stage to the issuer
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) i8_mbar_arrive_peer(ready_base + 8 * to);
            }
        }
    } else {
        // ---- epilogue: warps 4..7 the first 128 channels of the tile, 8..11 the second
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(I8W_REGS_EPI));
        const uint32_t quarter = warp & 3u, cbase = ((warp - 4) >> 2) * 128;
        const uint32_t tempty_base = i8_map_to_cta(bar_tempty, leader);
        uint32_t handover = 0;
        bool alive = true;
        for (uint32_t tile = unit0; alive && tile < num_tiles; tile += unit_stride) {
            uint32_t tx, ty;
            sgemm_tile_raster(tile, a.tiles_m, a.tiles_n, OPT_WGM, tx, ty);
            const uint32_t row = tx * 256 + rank * 128 + quarter * 32 + i8w_feature(lane), col0 = ty * 256 + cbase;
            // The running sum starts as beta * C, fetched while the tile's first chain is multiplied (taken one by one beside the stores, C
            // cost 4096 x 4096 in FP32 another 210 us).  The first part's sum has it.
            uint64_t sum2[64];
#pragma unroll
            for (int j = 0; j < 64; ++j) sum2[j] = 0ull;
            if (a.beta != 0.0f && part == 0) {
                const uint32_t row_first = tx * 256 + rank * 128 + quarter * 32;
                if (a.d_type == SGEMM_I8_FP32) i8w_add_c<SGEMM_I8_FP32>(sum2, a, row, row_first, col0);
                else if (a.d_type == SGEMM_I8_BF16) i8w_add_c<SGEMM_I8_BF16>(sum2, a, row, row_first, col0);
                else i8w_add_c<SGEMM_I8_FP16>(sum2, a, row, row_first, col0);
            }
            const uint64_t alpha2 = i8w_pair(a.alpha, a.alpha);
            for (uint32_t kb = kb_begin; kb < kb_end; kb += I8W_CHAIN, ++handover) {
                const uint32_t buf = handover & 1u, acc_phase = (handover >> 1) & 1u;
                alive = i8_wait_warp(waiter, bar_tfull + 8 * buf, acc_phase, 0x420u + buf, tile, kb);
                if (!alive) break;
                i8_fence_after();
#pragma unroll
                for (int cc = 0; cc < 16; ++cc) {
                    uint32_t r[8];
                    i8_tmem_ld8(tmem_base + ((quarter * 32u) << 16) + buf * 256 + cbase + cc * 8, r);
                    i8_tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        asm("{\n\t.reg .b64 t;\n\tmov.b64 t, {%1, %2};\n\tfma.rn.f32x2 %0, t, %3, %0;\n\t}"
                            : "+l"(sum2[cc * 4 + j]) : "r"(r[2 * j]), "r"(r[2 * j + 1]), "l"(alpha2));
                }
                i8_fence_before();
                __syncwarp();
                if (lane == 0) i8_mbar_arrive_peer(tempty_base + 8 * buf);
            }
            if (!alive) break;
            if (parts == 1) {
                if (a.d_type == SGEMM_I8_FP32) i8w_store_sums<SGEMM_I8_FP32>(sum2, a, row, col0);
                else if (a.d_type == SGEMM_I8_BF16) i8w_store_sums<SGEMM_I8_BF16>(sum2, a, row, col0);
                else i8w_store_sums<SGEMM_I8_FP16>(sum2, a, row, col0);
            } else {
                // (one tile per cluster.)  Every stage of the ring has been multiplied: the sums go over it, [column][row]
                const uint32_t mine = smem_base + (cbase * 128 + quarter * 32 + lane) * 4;
#pragma unroll
                for (int j = 0; j < 64; ++j) {
                    const float2 v = i8w_unpair(sum2[j]);
                    i8_sts(mine + (2 * j) * 512, __float_as_uint(v.x));
                    i8_sts(mine + (2 * j + 1) * 512, __float_as_uint(v.y));
                }
            }
        }
        if (parts > 1) {
            __syncwarp();
            i8_cluster_sync();
            if (!*abort_flag) {
                // eight warps, a column each at a time: lane l adds up four positions of it, 16 bytes per part.  The loads of two columns
                // over all parts are under way together (one after the other each would wait for the trip to a peer)
                uint32_t tx, ty;
                sgemm_tile_raster(unit0, a.tiles_m, a.tiles_n, OPT_WGM, tx, ty);
                const uint32_t row0 = tx * 256 + rank * 128 + lane * 4, from_peer = smem_base + lane * 16;
                const uint32_t first = 256u * part / parts, last = 256u * (part + 1) / parts;
                for (uint32_t j0 = first + warp - 4; j0 < last; j0 += 16) {
                    float4 v[2][4];
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int p = 0; p < 4; ++p)
                            v[u][p] = p < parts && j0 + 8 * u < last ? i8_ld_cluster4(i8_map_to_cta(from_peer + (j0 + 8 * u) * 512, 2 * p + rank))
                                                                     : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        float4 sum = v[u][0];
#pragma unroll
                        for (int p = 1; p < 4; ++p) {
                            sum.x += v[u][p].x; sum.y += v[u][p].y; sum.z += v[u][p].z; sum.w += v[u][p].w;
                        }
                        const float out[4] = {sum.x, sum.z, sum.y, sum.w};   // positions 0, 1, 2, 3 are features 0, 2, 1, 3
                        const uint32_t j = ty * 256 + j0 + 8 * u;
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (row0 + e < a.m && j < a.n && j0 + 8 * u < last) i8_store(a.d, row0 + e + (uint64_t)j * a.ldd, a.d_type, out[e]);
                    }
                }
            }
        }
    }
    __syncwarp();
    if (parts > 1 && (warp < 4 || warp >= 12)) i8_cluster_sync();   // the epilogue warps meet them at the barrier above
    i8_fence_before();
    i8_cluster_sync();   // no CTA of the cluster may release TMEM or exit while another can still reach into it
    if (warp == 1) {
        if (*abort_flag) i8_settle();
        i8_fence_after();
        i8_tmem_dealloc<2>(tmem_base, 512);
    }
}

// ------------------------------------------------------------ operands TMA cannot describe (and T = 0): FP32 multiply-adds
// 64 features x 64 channels per block, 16 tokens per step, 4 x 4 results per thread.
extern "C" __global__ void __launch_bounds__(I8_SIMT_THREADS) i8_wgrad_simt(const __grid_constant__ I8WgradArgs a) {
    __shared__ float tile_a[16][I8_SIMT_TILE], tile_g[16][I8_SIMT_TILE];
    sgemm_launch_dependents();
    sgemm_grid_dependency_wait();
    const uint32_t m0 = (blockIdx.x % a.tiles_m) * I8_SIMT_TILE, n0 = (blockIdx.x / a.tiles_m) * I8_SIMT_TILE;
    const uint32_t tm = threadIdx.x % 16, tn = threadIdx.x / 16, i = threadIdx.x % 64;
    float acc[4][4] = {};
    for (uint32_t t0 = 0; t0 < a.tokens; t0 += 16) {
        for (uint32_t r = threadIdx.x / 64; r < 16; r += I8_SIMT_THREADS / 64) {
            const uint32_t t = t0 + r;
            float v = 0.0f, g = 0.0f;
            if (t < a.tokens && m0 + i < a.m) {
                v = (float)a.q[(uint64_t)t * a.ldq + m0 + i] * a.scale[t];
                v = a.g_type == SGEMM_I8_BF16 ? __bfloat162float(__float2bfloat16_rn(v)) : __half2float(__float2half_rn(v));
            }
            if (t < a.tokens && n0 + i < a.n) g = i8_load(a.g, (uint64_t)t * a.ldg + n0 + i, a.g_type);
            tile_a[r][i] = v;
            tile_g[r][i] = g;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            float va[4], vg[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                va[e] = tile_a[r][tm + 16 * e];
                vg[e] = tile_g[r][tn + 16 * e];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int f = 0; f < 4; ++f) acc[e][f] = fmaf(va[e], vg[f], acc[e][f]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int f = 0; f < 4; ++f) {
            const uint32_t row = m0 + tm + 16 * e, col = n0 + tn + 16 * f;
            if (row >= a.m || col >= a.n) continue;
            float v = a.alpha * acc[e][f];
            if (a.beta != 0.0f) v = fmaf(a.beta, i8_load(a.c, row + (uint64_t)col * a.ldc, a.d_type), v);
            i8_store(a.d, row + (uint64_t)col * a.ldd, a.d_type, v);
        }
}
