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
// Roles, as in the in-kernel split of the FP32 kernel: a TMA producer brings a stage of I8W_BK tokens (raw int8 tile, G tile);
// four warps widen the raw tile into the A operand beside it; one thread of the pair's leader issues the MMAs; eight warps
// drain the accumulators.  CTA pairs (cta_group::2) work on 256 features x 256 channels: each CTA widens 128 features and
// stages 128 channels, so a widened element meets 256 channels and the widening (8192 elements a stage) hides beside the
// stage's 512 tensor cycles.
//
// Both operands are MN-major 16-bit tiles (a row of 128 bytes = 64 features or channels of one token, 128-byte swizzle,
// repeating unit 8 tokens: SBO = 1024; chunks of 64 features I8W_BK * 128 bytes apart: LBO); one MMA takes 16 tokens = 2048 bytes.
//
// The tensor core adds to its accumulator with truncation, so a long sum drifts toward zero: every I8W_CHAIN stages (the first two
// chains of a tile are twice as long) the issuer turns to the other TMEM buffer and the epilogue warps add the finished chain to
// a running sum in registers, rounding to nearest, in a fixed order.
//
// Few tiles and many tokens: S = 2 or 4 pairs of a cluster take S parts of the tokens of one tile.  Each leaves its sums in
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
#define I8W_REGS_WIDEN 56
#define I8W_REGS_EPI 208
static_assert(I8W_REGS_SMALL + I8W_REGS_WIDEN + 2 * I8W_REGS_EPI <= 4 * I8W_LAUNCH_REGS,
              "the register hand-over must not ask for more than the launch allocated");
static_assert(I8W_THREADS == 512 && I8W_SMEM <= 232448, "four groups of four warps, one CTA per SM");
static_assert(I8W_STAGES * I8W_STAGE_BYTES >= 128 * 256 * 4, "a part's sums must fit the drained ring");

// kind::f16 instruction descriptor: FP32 accumulator, A and B of one 16-bit type (0 = FP16, 1 = BF16), both MN-major, 256 x 256
__device__ __forceinline__ uint32_t i8w_idesc(uint32_t g_type) {
    const uint32_t fmt = g_type == SGEMM_I8_BF16 ? 1u : 0u;
    return (1u << 4) | (fmt << 7) | (fmt << 10) | (1u << 15) | (1u << 16) | ((256u >> 3) << 17) | ((256u >> 4) << 24);
}
__device__ __forceinline__ uint32_t i8w_chain_span(uint32_t blocks_done) { return blocks_done < 4u * I8W_CHAIN ? 2u * I8W_CHAIN : I8W_CHAIN; }

// two values to one word of G's type, round to nearest even
__device__ __forceinline__ uint32_t i8w_pack(float lo, float hi, uint32_t g_type) {
    uint32_t w;
    if (g_type == SGEMM_I8_BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    return w;
}

extern "C" __global__ void __launch_bounds__(I8W_THREADS, 1)
i8_wgrad(const __grid_constant__ I8WgradArgs a, const __grid_constant__ I8TensorMap map_q, const __grid_constant__ I8TensorMap map_g) {
    extern __shared__ uint8_t i8_smem_raw[];
    const uint32_t smem_base = (i8_smem_u32(i8_smem_raw) + 1023u) & ~1023u;
    uint8_t *generic_base = i8_smem_raw + (smem_base - i8_smem_u32(i8_smem_raw));
    // a stage: [widened A | G | raw]; barrier block: full[S] | empty[S] | ready[S] | tmem_full[2] | tmem_empty[2] | base | abort
    const uint32_t bar_full = smem_base + I8W_STAGES * I8W_STAGE_BYTES, bar_empty = bar_full + 8 * I8W_STAGES;
    const uint32_t bar_ready = bar_empty + 8 * I8W_STAGES, bar_tfull = bar_ready + 8 * I8W_STAGES, bar_tempty = bar_tfull + 16;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(generic_base + I8W_STAGES * I8W_STAGE_BYTES + 24 * I8W_STAGES + 32);
    volatile uint32_t *abort_flag = tmem_slot + 1;
    static_assert(24 * I8W_STAGES + 32 + 8 <= 256, "barrier block size");
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const I8Wait waiter{abort_flag, a.status, I8_TIMEOUT_NS};
    // the cluster holds S pairs; pair z takes the z-th part of the tokens, its even CTA leads
    const uint32_t cluster_rank = i8_cluster_rank(), parts = i8_cluster_size() / 2, part = cluster_rank / 2, rank = cluster_rank & 1u;
    const uint32_t leader = cluster_rank & ~1u, peer = cluster_rank | 1u;
    const uint32_t unit0 = blockIdx.x / (2 * parts), unit_stride = gridDim.x / (2 * parts);
    const uint32_t num_tiles = a.tiles_m * a.tiles_n;
    const uint32_t blocks = (a.tokens + I8W_BK - 1) / I8W_BK;
    const uint32_t kb_begin = (uint32_t)((uint64_t)blocks * part / parts), kb_end = (uint32_t)((uint64_t)blocks * (part + 1) / parts);

    if (threadIdx.x == 0) {
        for (int s = 0; s < I8W_STAGES; ++s) {
            i8_mbar_init(bar_full + 8 * s, 1);
            i8_mbar_init(bar_empty + 8 * s, 1);
            i8_mbar_init(bar_ready + 8 * s, 4 * 2);
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
            if (lane == 0) {   // ---- TMA producer: each CTA's loads report to its own "full" barrier (it widens what it loaded)
                uint32_t stage = 0, phase = 0;
                bool alive = true;
                for (uint32_t tile = unit0; alive && tile < num_tiles; tile += unit_stride) {
                    uint32_t tx, ty;
                    sgemm_tile_raster(tile, a.tiles_m, a.tiles_n, OPT_WGM, tx, ty);
                    const int32_t m0 = (int32_t)(tx * 256 + rank * 128), n0 = (int32_t)(ty * 256 + rank * 128);
                    for (uint32_t kb = kb_begin; kb < kb_end; ++kb) {
                        if (!i8_wait(waiter, bar_empty + 8 * stage, phase ^ 1u, 0x120u + stage, tile, kb)) { alive = false; break; }
                        const uint32_t sa = smem_base + stage * I8W_STAGE_BYTES, sg = sa + I8W_OP_BYTES, raw = sg + I8W_OP_BYTES;
                        const uint32_t full = bar_full + 8 * stage;
                        const int32_t t0 = (int32_t)(kb * I8W_BK);
                        i8_mbar_expect_tx(full, I8W_RAW_BYTES + I8W_OP_BYTES);
                        i8_tma_load(raw, &map_q, full, m0, t0);
                        i8_tma_load(sg, &map_g, full, n0, t0);
                        i8_tma_load(sg + I8W_CHUNK_BYTES, &map_g, full, n0 + 64, t0);
                        if (++stage == I8W_STAGES) { stage = 0; phase ^= 1u; }
                    }
                }
            }
        } else if (warp == 1) {
            if (lane == 0 && rank == 0) {   // ---- MMA issuer
                const uint32_t idesc = i8w_idesc(a.g_type);
                uint32_t stage = 0, phase = 0, handover = 0;
                bool alive = true;
                for (uint32_t tile = unit0; alive && tile < num_tiles; tile += unit_stride) {
                    for (uint32_t kb = kb_begin; alive && kb < kb_end;) {
                        const uint32_t buf = handover & 1u, acc_phase = (handover >> 1) & 1u;
                        if (!i8_wait(waiter, bar_tempty + 8 * buf, acc_phase ^ 1u, 0x220u + buf, tile, kb)) { alive = false; break; }
                        i8_fence_after();
                        const uint32_t chain_begin = kb, chain_end = min(kb_end, kb + i8w_chain_span(kb - kb_begin));
                        for (; kb < chain_end; ++kb) {
                            if (!i8_wait(waiter, bar_ready + 8 * stage, phase, 0x320u + stage, tile, kb)) { alive = false; break; }
                            i8_fence_after();
                            const uint32_t sa = smem_base + stage * I8W_STAGE_BYTES, sg = sa + I8W_OP_BYTES;
#pragma unroll
                            for (int kk = 0; kk < I8W_BK / 16; ++kk)
                                i8_mma_f16_pair(tmem_base + buf * 256, i8_smem_desc(sa + kk * 2048, I8W_CHUNK_BYTES, 1024),
                                                i8_smem_desc(sg + kk * 2048, I8W_CHUNK_BYTES, 1024), idesc, (kb == chain_begin && kk == 0) ? 0u : 1u);
                            i8_commit<2>(bar_empty + 8 * stage, peer);
                            if (++stage == I8W_STAGES) { stage = 0; phase ^= 1u; }
                        }
                        if (alive) i8_commit<2>(bar_tfull + 8 * buf, peer);
                        ++handover;
                    }
                }
            }
        }
    } else if (warp >= 12) {
        // ---- widening: thread t of 128 takes token t / 8 (and + 16, 32, 48), features 16 (t % 8) .. + 15
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(I8W_REGS_WIDEN));
        const uint32_t t = threadIdx.x - 384, unit = t & 7u, tok = t >> 3;
        const uint32_t ready_base = i8_map_to_cta(bar_ready, leader);
        // the two 16-byte halves of a thread's 16 values; lanes of the second chunk write them in the other order, so that the
        // eight lanes of a token hit eight different units of the swizzled rows
        const uint32_t chunk = unit >> 2, j0 = (unit & 3u) * 2 + chunk, j1 = (unit & 3u) * 2 + (chunk ^ 1u);
        uint32_t stage = 0, phase = 0;
        bool alive = true;
        for (uint32_t tile = unit0; alive && tile < num_tiles; tile += unit_stride) {
            for (uint32_t kb = kb_begin; kb < kb_end; ++kb) {
                float s[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t token = kb * I8W_BK + tok + 16 * i;
                    s[i] = token < a.tokens ? __ldg(a.scale + token) : 0.0f;   // beyond the last token both tiles are zero-filled
                }
                alive = __all_sync(0xffffffffu, i8_wait(waiter, bar_full + 8 * stage, phase, 0x520u + stage, tile, kb));
                if (!alive) break;
                uint8_t *sa = generic_base + stage * I8W_STAGE_BYTES;
                const uint8_t *raw = sa + 2 * I8W_OP_BYTES;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t row = tok + 16 * i;
                    const uint4 w = *reinterpret_cast<const uint4 *>(raw + row * 128 + unit * 16);
                    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
                    uint32_t o[8];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        float v[4];
                        i8_widen4(words[k], v);
                        o[2 * k] = i8w_pack(v[0] * s[i], v[1] * s[i], a.g_type);
                        o[2 * k + 1] = i8w_pack(v[2] * s[i], v[3] * s[i], a.g_type);
                    }
                    uint8_t *dst = sa + chunk * I8W_CHUNK_BYTES + row * 128;
                    const uint4 lo = make_uint4(o[0], o[1], o[2], o[3]), hi = make_uint4(o[4], o[5], o[6], o[7]);
                    *reinterpret_cast<uint4 *>(dst + ((j0 ^ (row & 7u)) << 4)) = chunk ? hi : lo;
                    *reinterpret_cast<uint4 *>(dst + ((j1 ^ (row & 7u)) << 4)) = chunk ? lo : hi;
                }
                // generic-proxy writes -> visible to the tensor core (async proxy), then hand the stage to the issuer
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) i8_mbar_arrive_cluster(ready_base + 8 * stage);
                if (++stage == I8W_STAGES) { stage = 0; phase ^= 1u; }
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
            const uint32_t row = tx * 256 + rank * 128 + quarter * 32 + lane, col0 = ty * 256 + cbase;
            uint64_t sum2[64];   // the running sum: two columns per 64-bit register pair, packed FP32 adds
#pragma unroll
            for (int j = 0; j < 64; ++j) sum2[j] = 0ull;
            for (uint32_t kb = kb_begin; kb < kb_end; kb += i8w_chain_span(kb - kb_begin), ++handover) {
                const uint32_t buf = handover & 1u, acc_phase = (handover >> 1) & 1u;
                alive = __all_sync(0xffffffffu, i8_wait(waiter, bar_tfull + 8 * buf, acc_phase, 0x420u + buf, tile, kb));
                if (!alive) break;
                i8_fence_after();
#pragma unroll
                for (int cc = 0; cc < 8; ++cc) {
                    uint32_t r[16];
                    i8_tmem_ld16(tmem_base + ((quarter * 32u) << 16) + buf * 256 + cbase + cc * 16, r);
                    i8_tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        asm("{\n\t.reg .b64 t;\n\tmov.b64 t, {%1, %2};\n\tadd.rn.f32x2 %0, %0, t;\n\t}"
                            : "+l"(sum2[cc * 8 + j]) : "r"(r[2 * j]), "r"(r[2 * j + 1]));
                }
                i8_fence_before();
                __syncwarp();
                if (lane == 0) i8_mbar_arrive_cluster(tempty_base + 8 * buf);
            }
            if (!alive) break;
            if (parts == 1) {
                const bool use_c = a.beta != 0.0f;
#pragma unroll
                for (int j = 0; j < 128; ++j) {
                    const uint32_t col = col0 + j;
                    float lo, hi;
                    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(sum2[j / 2]));
                    float v = a.alpha * ((j & 1) ? hi : lo);
                    if (row < a.m && col < a.n) {
                        if (use_c) v = fmaf(a.beta, i8_load(a.c, row + (uint64_t)col * a.ldc, a.d_type), v);
                        i8_store(a.d, row + (uint64_t)col * a.ldd, a.d_type, v);
                    }
                }
            } else {
                // (one tile per cluster.)  Every stage of the ring has been multiplied: the sums go over it, [column][row]
                float *mine = reinterpret_cast<float *>(generic_base) + cbase * 128 + quarter * 32 + lane;
#pragma unroll
                for (int j = 0; j < 64; ++j) {
                    float lo, hi;
                    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(sum2[j]));
                    mine[(2 * j) * 128] = lo;
                    mine[(2 * j + 1) * 128] = hi;
                }
            }
        }
    }
    __syncwarp();
    if (parts > 1) {
        i8_cluster_sync();
        if (!*abort_flag && warp >= 4 && warp < 12) {
            // eight warps: quarter w % 4 of the rows, every second of this part's columns
            uint32_t tx, ty;
            sgemm_tile_raster(unit0, a.tiles_m, a.tiles_n, OPT_WGM, tx, ty);
            const uint32_t local = (warp & 3u) * 32 + lane, row = tx * 256 + rank * 128 + local;
            for (uint32_t col = part * 2 + ((warp - 4) >> 2); col < 256; col += 2 * parts) {
                float v = 0.0f;
                for (uint32_t p = 0; p < parts; ++p)
                    v += __uint_as_float(i8_ld_cluster(i8_map_to_cta(smem_base + (col * 128 + local) * 4, 2 * p + rank)));
                const uint32_t j = ty * 256 + col;
                if (row < a.m && j < a.n) {
                    v *= a.alpha;
                    if (a.beta != 0.0f) v = fmaf(a.beta, i8_load(a.c, row + (uint64_t)j * a.ldc, a.d_type), v);
                    i8_store(a.d, row + (uint64_t)j * a.ldd, a.d_type, v);
                }
            }
        }
        __syncwarp();
    }
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
