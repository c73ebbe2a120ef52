// ---------------------------------------------------------------------------------------------
// Linear layer on 8-bit integers (tcgen05 kind::i8, int32 accumulators in TMEM).
//
//   Y[i, j] = fp32(sum_k W[k, i] * X[k, j]) * sx[j] * sw[i] (+ bias[i])        i < M channels, j < N tokens
//
// W is K x M and X is K x N, both column-major with K contiguous (the transposed-A layout of the FP32 and 16-bit kernels);
// Y is M x N column-major: a token's channels are contiguous.  The integer sum is exact (K <= 131071), so it does not
// depend on the tile, the split of K or the order of anything; it is converted to FP32 once (2^-24) and scaled in FP32, then
// rounded once to Y's type.
//
// Operand tiles: K-major rows of 128 int8 under the 128-byte swizzle (SBO = 1024), one MMA takes 32 bytes of K of every
// row, so a stage of 128 k is four MMAs.
//
// Channels lie on the MMA's M axis for every kernel here: a TMEM lane is a channel, so the 32 lanes of an epilogue warp write 32
// consecutive channels of one token (64 bytes of a 16-bit Y, whole sectors) straight from registers, for any base and
// leading dimension of Y, and a lane holds its channel's scale and bias in two registers.
//
//   generated_gemm     CTA pair (cta_group::2) on 256 channels x I8_BN tokens, persistent, two accumulators in TMEM: the
//                      epilogue of a tile runs beside the main loop of the next one.  A pair reads each operand tile once
//                      per 256 rows of the other, half of what two single CTAs would, which is what lets shared memory
//                      feed the 8-bit rate.
//   i8_linear_half     the same on 256 channels x 128 tokens, for problems whose 256 x 256 tiles leave half of the SMs idle.
//   i8_linear_few_TN   one CTA on 128 channels x TN tokens and one part of K; the CTAs of a cluster hold the parts of one tile
//                      and add their int32 partials through distributed shared memory.  For few tokens the layer is bound
//                      by reading W once: small tiles and a cut K put every SM on it, without a workspace in global
//                      memory, without a second launch and without atomics.
//   generated_gemm_simt  operands TMA cannot describe: 64 x 64 tiles with dp4a.
// ---------------------------------------------------------------------------------------------
#ifndef I8_BN
#error "the generator defines I8_BN (tokens per tile), I8_STAGES and OPT_WGM"
#endif

// kind::i8 instruction descriptor: int32 accumulator [4,6) = 2, signed A and B [7,10) = [10,13) = 1, both K-major,
// N>>3 at [17,23), M>>4 at [24,29)
#define I8_IDESC(m, n) ((2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)((n) >> 3) << 17) | ((uint32_t)((m) >> 4) << 24))

struct I8LinearArgs {
    const int8_t *w;
    const float *sw;
    const int8_t *x;
    const float *sx;
    const float *bias;    // or NULL
    void *y;
    uint32_t *status;
    uint32_t m, n, k, ldw, ldx, ldy;
    uint32_t y_type;
    uint32_t tiles_m, tiles_n;
};

// Issue the four MMAs of one stage: a step of 32 bytes of K inside the swizzled rows.
template <int GROUP>
__device__ __forceinline__ void i8_stage_mma(uint32_t d_tmem, uint64_t desc_w, uint64_t desc_x, uint32_t idesc, bool first) {
#pragma unroll
    for (int kk = 0; kk < I8_BK / 32; ++kk)
        i8_mma_s8<GROUP>(d_tmem, desc_w + kk * 2, desc_x + kk * 2, idesc, (first && kk == 0) ? 0u : 1u);
}

// One TMEM lane's (channel's) accumulators of COLS tokens -> Y.  `sx` of token col0 + lane sits in lane `lane`.
template <uint32_t TYPE, int COLS>
__device__ __forceinline__ void i8_store_columns(const uint32_t (&acc)[COLS], const I8LinearArgs &a, uint32_t channel, uint32_t col0,
                                                 float sx_lane, float sw, float bias) {
    using E = I8Elem<TYPE>;
    using T = typename E::type;
    T *y = static_cast<T *>(a.y) + channel + (uint64_t)col0 * a.ldy;
    const bool row_ok = channel < a.m;
    const uint32_t cols = a.n > col0 ? a.n - col0 : 0u;
    if (cols >= COLS) {
#pragma unroll
        for (int j = 0; j < COLS; ++j) {
            const float v = fmaf((float)(int32_t)acc[j] * __shfl_sync(0xffffffffu, sx_lane, j), sw, bias);
            if (row_ok) *y = E::put(v);
            y += a.ldy;
        }
    } else {
#pragma unroll
        for (int j = 0; j < COLS; ++j) {
            const float v = fmaf((float)(int32_t)acc[j] * __shfl_sync(0xffffffffu, sx_lane, j), sw, bias);
            if (row_ok && j < cols) *y = E::put(v);
            y += a.ldy;
        }
    }
}
template <int COLS>
__device__ __forceinline__ void i8_store_columns_any(const uint32_t (&acc)[COLS], const I8LinearArgs &a, uint32_t channel,
                                                     uint32_t col0, float sx_lane, float sw, float bias) {
    if (a.y_type == SGEMM_I8_BF16) i8_store_columns<SGEMM_I8_BF16, COLS>(acc, a, channel, col0, sx_lane, sw, bias);
    else if (a.y_type == SGEMM_I8_FP16) i8_store_columns<SGEMM_I8_FP16, COLS>(acc, a, channel, col0, sx_lane, sw, bias);
    else i8_store_columns<SGEMM_I8_FP32, COLS>(acc, a, channel, col0, sx_lane, sw, bias);
}

// ------------------------------------------------------------------------------- many tokens: CTA pairs
#define I8_W_BYTES (I8_BM * I8_BK)

template <int BN, int STAGES>
__device__ __forceinline__ void i8_linear_pair(const I8LinearArgs &a, const I8TensorMap &map_w, const I8TensorMap &map_x) {
    constexpr uint32_t BN_CTA = BN / 2;              // tokens of a tile this CTA keeps in shared memory
    constexpr uint32_t STAGE_BYTES = I8_W_BYTES + BN_CTA * I8_BK;
    constexpr uint32_t EPI_COLS = BN / 2;            // columns one of the two epilogue warps of a lane quarter drains
    constexpr uint32_t TMEM_COLS = 2 * BN <= 128 ? 128 : 2 * BN <= 256 ? 256 : 512;
    static_assert(BN % 64 == 0 && BN <= 256, "two accumulators in TMEM, whole 32-column chunks per epilogue warp");
    static_assert(I8_PAIR_SMEM(BN, STAGES) <= 232448, "shared memory budget of one CTA");
    static_assert(16 * STAGES + 32 + 8 <= 256, "barrier block size");
    extern __shared__ uint8_t i8_smem_raw[];
    const uint32_t smem_base = (i8_smem_u32(i8_smem_raw) + 1023u) & ~1023u;
    const uint32_t bar_base = smem_base + STAGES * STAGE_BYTES;
    // barrier block: full[S] | empty[S] | tmem_full[2] | tmem_empty[2] | tmem base (u32) | abort (u32)
    const uint32_t bar_full = bar_base, bar_empty = bar_base + 8 * STAGES;
    const uint32_t bar_tfull = bar_base + 16 * STAGES, bar_tempty = bar_tfull + 16;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(i8_smem_raw + (bar_tempty + 16 - i8_smem_u32(i8_smem_raw)));
    volatile uint32_t *abort_flag = tmem_slot + 1;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const I8Wait waiter{abort_flag, a.status, I8_TIMEOUT_NS};
    const uint32_t rank = i8_cluster_rank();
    const uint32_t unit0 = blockIdx.x / 2, unit_stride = gridDim.x / 2;
    const uint32_t num_tiles = a.tiles_m * a.tiles_n;
    const uint32_t kbs = (a.k + I8_BK - 1) / I8_BK;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            i8_mbar_init(bar_full + 8 * s, 1);
            i8_mbar_init(bar_empty + 8 * s, 1);
        }
        for (int i = 0; i < 2; ++i) {
            i8_mbar_init(bar_tfull + 8 * i, 1);
            i8_mbar_init(bar_tempty + 8 * i, 8 * 2);
        }
        *abort_flag = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        i8_prefetch_map(&map_w);
        i8_prefetch_map(&map_x);
    }
    if (warp == 1) i8_tmem_alloc<2>(i8_smem_u32(tmem_slot), TMEM_COLS);
    i8_fence_before();
    i8_cluster_sync();   // the peer's barriers must be initialised before anything is signalled to them
    i8_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    sgemm_launch_dependents();
    sgemm_grid_dependency_wait();

    if (warp == 0) {   // ---- TMA producer: both CTAs' loads report to the leader's "full" barrier
        uint32_t stage = 0, phase = 0;
        bool alive = true;
        const uint32_t full_base = i8_map_to_cta(bar_full, 0u);
        for (uint32_t tile = unit0; alive && tile < num_tiles; tile += unit_stride) {
            uint32_t tx, ty;
            sgemm_tile_raster(tile, a.tiles_m, a.tiles_n, OPT_WGM, tx, ty);
            const int32_t m0 = (int32_t)(tx * 256 + rank * I8_BM), n0 = (int32_t)(ty * BN + rank * BN_CTA);
            for (uint32_t kb = 0; kb < kbs; ++kb) {
                if (!i8_wait_warp(waiter, bar_empty + 8 * stage, phase ^ 1u, 0x100u + stage, tile, kb)) { alive = false; break; }
                const uint32_t sw = smem_base + stage * STAGE_BYTES, sx = sw + I8_W_BYTES;
                if (i8_elect()) {
                    if (rank == 0) i8_mbar_expect_tx(bar_full + 8 * stage, 2 * STAGE_BYTES);
                    i8_tma_load_pair(sw, &map_w, full_base + 8 * stage, (int32_t)(kb * I8_BK), m0);
                    i8_tma_load_pair(sx, &map_x, full_base + 8 * stage, (int32_t)(kb * I8_BK), n0);
                }
                if (++stage == STAGES) { stage = 0; phase ^= 1u; }
            }
        }
    } else if (warp == 1) {
        if (rank == 0) {   // ---- MMA issuer
            uint32_t stage = 0, phase = 0, handover = 0;
            bool alive = true;
            const uint64_t desc_w0 = i8_smem_desc(smem_base, 16, 1024), desc_x0 = i8_smem_desc(smem_base + I8_W_BYTES, 16, 1024);
            uint64_t desc_w = desc_w0, desc_x = desc_x0;
            for (uint32_t tile = unit0; alive && tile < num_tiles; tile += unit_stride, ++handover) {
                const uint32_t buf = handover & 1u, acc_phase = (handover >> 1) & 1u;
                if (!i8_wait_warp(waiter, bar_tempty + 8 * buf, acc_phase ^ 1u, 0x200u + buf, tile, 0)) break;
                i8_fence_after();
                for (uint32_t kb = 0; kb < kbs; ++kb) {
                    if (!i8_wait_warp(waiter, bar_full + 8 * stage, phase, 0x300u + stage, tile, kb)) { alive = false; break; }
                    i8_fence_after();
                    if (i8_elect()) {
                        i8_stage_mma<2>(tmem_base + buf * BN, desc_w, desc_x, I8_IDESC(256, BN), kb == 0);
                        i8_commit<2>(bar_empty + 8 * stage, 3);
                        if (kb + 1 == kbs) i8_commit<2>(bar_tfull + 8 * buf, 3);
                    }
                    desc_w += STAGE_BYTES / 16;
                    desc_x += STAGE_BYTES / 16;
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                        desc_w = desc_w0;
                        desc_x = desc_x0;
                    }
                }
            }
        }
    } else if (warp >= 4) {   // ---- epilogue: warps 4..7 the first half of the tile's tokens, 8..11 the second
        const uint32_t quarter = warp & 3u, cbase = ((warp - 4) >> 2) * EPI_COLS;
        const uint32_t tempty_base = i8_map_to_cta(bar_tempty, 0u);
        uint32_t handover = 0;
        for (uint32_t tile = unit0; tile < num_tiles; tile += unit_stride, ++handover) {
            uint32_t tx, ty;
            sgemm_tile_raster(tile, a.tiles_m, a.tiles_n, OPT_WGM, tx, ty);
            const uint32_t channel = tx * 256 + rank * I8_BM + quarter * 32 + lane, col0 = ty * BN + cbase;
            const float sw = channel < a.m ? __ldg(a.sw + channel) : 0.0f;
            const float bias = a.bias && channel < a.m ? __ldg(a.bias + channel) : 0.0f;
            float sx[EPI_COLS / 32];
#pragma unroll
            for (int c = 0; c < EPI_COLS / 32; ++c) sx[c] = col0 + c * 32 + lane < a.n ? __ldg(a.sx + col0 + c * 32 + lane) : 0.0f;
            const uint32_t buf = handover & 1u, acc_phase = (handover >> 1) & 1u;
            if (!i8_wait_warp(waiter, bar_tfull + 8 * buf, acc_phase, 0x400u + buf, tile, 0)) break;
            i8_fence_after();
#pragma unroll
            for (int c = 0; c < EPI_COLS / 32; ++c) {
                uint32_t acc[32];
                i8_tmem_ld32(tmem_base + ((quarter * 32u) << 16) + buf * BN + cbase + c * 32, acc);
                i8_tmem_ld_wait();
                if (c + 1 == EPI_COLS / 32) {   // the buffer is read: hand it back before the stores
                    i8_fence_before();
                    __syncwarp();
                    if (lane == 0) i8_mbar_arrive_peer(tempty_base + 8 * buf);
                }
                i8_store_columns_any<32>(acc, a, channel, col0 + c * 32, sx[c], sw, bias);
            }
        }
    }
    i8_fence_before();
    __syncwarp();
    i8_cluster_sync();   // neither CTA may release TMEM or exit while the other can still reach into it
    if (warp == 1) {
        if (*abort_flag) i8_settle();
        i8_fence_after();
        i8_tmem_dealloc<2>(tmem_base, TMEM_COLS);
    }
}
#define I8_PAIR_KERNEL(NAME, BN, STAGES)                                                                            \
    extern "C" __global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(I8_PAIR_THREADS, 1)                      \
    NAME(const __grid_constant__ I8LinearArgs a, const __grid_constant__ I8TensorMap map_w, const __grid_constant__ I8TensorMap map_x) { \
        i8_linear_pair<BN, STAGES>(a, map_w, map_x);                                                                \
    }
I8_PAIR_KERNEL(generated_gemm, I8_BN, I8_STAGES)
I8_PAIR_KERNEL(i8_linear_half, I8_HALF_BN, I8_HALF_STAGES)

// ---------------------------------------------------------------- few tokens: K cut over the CTAs of a cluster
// Cluster of S = 1, 2, 4 or 8 CTAs per tile (a launch attribute).  CTA r takes the r-th of S even parts of K's stages.  With S > 1
// each CTA leaves its int32 partial in its own shared memory (over the drained ring), [token][channel], and after a
// cluster barrier CTA r adds up tokens r, r + S, ... of all S partials.
template <int TN, int STAGES>
__device__ __forceinline__ void i8_linear_few(const I8LinearArgs &a, const I8TensorMap &map_w, const I8TensorMap &map_x) {
    constexpr uint32_t X_BYTES = TN * I8_BK, STAGE_BYTES = I8_W_BYTES + X_BYTES;
    constexpr uint32_t TMEM_COLS = TN < 32 ? 32 : TN;
    constexpr int CHUNK = TN < 32 ? TN : 32;
    static_assert(STAGES * STAGE_BYTES >= TN * I8_BM * 4, "the partial tile must fit the ring");
    static_assert(16 * STAGES + 16 <= 256, "barrier block size");
    extern __shared__ uint8_t i8_few_smem_raw[];
    const uint32_t smem_base = (i8_smem_u32(i8_few_smem_raw) + 1023u) & ~1023u;
    const uint32_t bar_full = smem_base + STAGES * STAGE_BYTES, bar_empty = bar_full + 8 * STAGES, bar_done = bar_empty + 8 * STAGES;
    uint8_t *generic_base = i8_few_smem_raw + (smem_base - i8_smem_u32(i8_few_smem_raw));
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(generic_base + STAGES * STAGE_BYTES + 16 * STAGES + 8);
    volatile uint32_t *abort_flag = tmem_slot + 1;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const I8Wait waiter{abort_flag, a.status, I8_TIMEOUT_NS};
    const uint32_t parts = i8_cluster_size(), rank = i8_cluster_rank(), tile = blockIdx.x / parts;
    const uint32_t tx = tile % a.tiles_m, ty = tile / a.tiles_m;
    const uint32_t kbs = (a.k + I8_BK - 1) / I8_BK;
    const uint32_t kb_begin = (uint32_t)((uint64_t)kbs * rank / parts), kb_end = (uint32_t)((uint64_t)kbs * (rank + 1) / parts);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            i8_mbar_init(bar_full + 8 * s, 1);
            i8_mbar_init(bar_empty + 8 * s, 1);
        }
        i8_mbar_init(bar_done, 1);
        *abort_flag = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        i8_prefetch_map(&map_w);
        i8_prefetch_map(&map_x);
    }
    if (warp == 1) i8_tmem_alloc<1>(i8_smem_u32(tmem_slot), TMEM_COLS);
    i8_fence_before();
    __syncthreads();
    i8_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    sgemm_launch_dependents();
    sgemm_grid_dependency_wait();

    if (warp == 0) {
        uint32_t stage = 0, phase = 0;
        for (uint32_t kb = kb_begin; kb < kb_end; ++kb) {
            if (!i8_wait_warp(waiter, bar_empty + 8 * stage, phase ^ 1u, 0x110u + stage, tile, kb)) break;
            const uint32_t sw = smem_base + stage * STAGE_BYTES, full = bar_full + 8 * stage;
            if (i8_elect()) {
                i8_mbar_expect_tx(full, STAGE_BYTES);
                i8_tma_load(sw, &map_w, full, (int32_t)(kb * I8_BK), (int32_t)(tx * I8_BM));
                i8_tma_load(sw + I8_W_BYTES, &map_x, full, (int32_t)(kb * I8_BK), (int32_t)(ty * TN));
            }
            if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
    } else if (warp == 1) {
        uint32_t stage = 0, phase = 0;
        for (uint32_t kb = kb_begin; kb < kb_end; ++kb) {
            if (!i8_wait_warp(waiter, bar_full + 8 * stage, phase, 0x310u + stage, tile, kb)) break;
            i8_fence_after();
            const uint64_t desc_w = i8_smem_desc(smem_base, 16, 1024) + stage * (STAGE_BYTES / 16);
            if (i8_elect()) {
                i8_stage_mma<1>(tmem_base, desc_w, desc_w + I8_W_BYTES / 16, I8_IDESC(I8_BM, TN), kb == kb_begin);
                i8_commit<1>(bar_empty + 8 * stage, 0);
                if (kb + 1 == kb_end) i8_commit<1>(bar_done, 0);
            }
            if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
    }
    __syncwarp();
    const uint32_t channel = tx * I8_BM + warp * 32 + lane, col_first = ty * TN;
    const float sw = channel < a.m ? __ldg(a.sw + channel) : 0.0f;
    const float bias = a.bias && channel < a.m ? __ldg(a.bias + channel) : 0.0f;
    const bool empty = kb_begin == kb_end;   // more parts than stages: this CTA's partial is zero
    const bool done = empty || i8_wait_warp(waiter, bar_done, 0u, 0x410u, tile, 0);
    i8_fence_after();
    const uint32_t cols = min((uint32_t)TN, a.n - col_first);
    if (done) {
#pragma unroll
        for (int c = 0; c < TN / CHUNK; ++c) {
            if (c * CHUNK < cols) {
                uint32_t acc[CHUNK];
                if constexpr (CHUNK == 32) i8_tmem_ld32(tmem_base + ((warp * 32u) << 16) + c * CHUNK, acc);
                else i8_tmem_ld16(tmem_base + ((warp * 32u) << 16) + c * CHUNK, acc);
                i8_tmem_ld_wait();
                if (parts == 1) {
                    const float sx = col_first + c * CHUNK + lane < a.n && lane < CHUNK ? __ldg(a.sx + col_first + c * CHUNK + lane) : 0.0f;
                    i8_store_columns_any<CHUNK>(acc, a, channel, col_first + c * CHUNK, sx, sw, bias);
                } else {
                    const uint32_t part = smem_base + (c * CHUNK * I8_BM + threadIdx.x) * 4;
#pragma unroll
                    for (int j = 0; j < CHUNK; ++j)
                        if (c * CHUNK + j < cols) i8_sts(part + j * (I8_BM * 4), empty ? 0u : acc[j]);
                }
            }
        }
    }
    if (parts > 1) {
        __syncwarp();
        i8_cluster_sync();
        if (done) {
            // a warp takes a token, a lane four channels of it (16 bytes of each partial); all parts of two tokens are under way together:
            // a load from a peer is a long trip
            const uint32_t first = tx * I8_BM + lane * 4;
            float sw4[4], bias4[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sw4[e] = first + e < a.m ? __ldg(a.sw + first + e) : 0.0f;
                bias4[e] = a.bias && first + e < a.m ? __ldg(a.bias + first + e) : 0.0f;
            }
            for (uint32_t j0 = rank + warp * parts; j0 < cols; j0 += 8 * parts) {
                uint4 v[2][8];
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int p = 0; p < 8; ++p)
                        v[u][p] = p < parts && j0 + u * 4 * parts < cols
                                      ? i8_ld_cluster4u(i8_map_to_cta(smem_base + (j0 + u * 4 * parts) * (I8_BM * 4) + lane * 16, p)) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint32_t j = j0 + u * 4 * parts;
                    if (j < cols) {
                        uint32_t sum[4] = {0u, 0u, 0u, 0u};
#pragma unroll
                        for (int p = 0; p < 8; ++p) {
                            sum[0] += v[u][p].x; sum[1] += v[u][p].y; sum[2] += v[u][p].z; sum[3] += v[u][p].w;
                        }
                        const float sx = __ldg(a.sx + col_first + j);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (first + e < a.m)
                                i8_store(a.y, first + e + (uint64_t)(col_first + j) * a.ldy, a.y_type, fmaf((float)(int32_t)sum[e] * sx, sw4[e], bias4[e]));
                    }
                }
            }
        }
        __syncwarp();
        i8_cluster_sync();   // the peers may still be reading this CTA's partial
    }
    i8_fence_before();
    __syncthreads();
    if (warp == 1) {
        if (*abort_flag) i8_settle();
        i8_fence_after();
        i8_tmem_dealloc<1>(tmem_base, TMEM_COLS);
    }
}
#define I8_FEW_KERNEL(TN)                                                                                          \
    extern "C" __global__ void __launch_bounds__(I8_FEW_THREADS)                                                   \
    i8_linear_few_##TN(const __grid_constant__ I8LinearArgs a, const __grid_constant__ I8TensorMap map_w,          \
                       const __grid_constant__ I8TensorMap map_x) {                                                \
        i8_linear_few<TN, I8_FEW_STAGES_##TN>(a, map_w, map_x);                                                    \
    }
I8_FEW_KERNEL(16)
I8_FEW_KERNEL(32)
I8_FEW_KERNEL(64)
I8_FEW_KERNEL(128)

// ------------------------------------------------------------ operands TMA cannot describe: dp4a
// 64 channels x 64 tokens per block, 64 k per step, 4 x 4 results per thread.  Rows start at any byte: a row's bytes are
// loaded one by one, coalesced along k, and packed through shared memory.
extern "C" __global__ void __launch_bounds__(I8_SIMT_THREADS) generated_gemm_simt(const __grid_constant__ I8LinearArgs a) {
    __shared__ __align__(16) int8_t tile_w[I8_SIMT_TILE][68], tile_x[I8_SIMT_TILE][68];   // 17 words a row: no bank conflicts
    sgemm_launch_dependents();
    sgemm_grid_dependency_wait();
    const uint32_t m0 = (blockIdx.x % a.tiles_m) * I8_SIMT_TILE, n0 = (blockIdx.x / a.tiles_m) * I8_SIMT_TILE;
    const uint32_t tm = threadIdx.x % 16, tn = threadIdx.x / 16;
    int32_t acc[4][4] = {};
    for (uint32_t k0 = 0; k0 < a.k; k0 += 64) {
        const uint32_t kk = threadIdx.x % 64;
        for (uint32_t r = threadIdx.x / 64; r < I8_SIMT_TILE; r += I8_SIMT_THREADS / 64) {
            const bool k_ok = k0 + kk < a.k;
            tile_w[r][kk] = k_ok && m0 + r < a.m ? a.w[(uint64_t)(m0 + r) * a.ldw + k0 + kk] : (int8_t)0;
            tile_x[r][kk] = k_ok && n0 + r < a.n ? a.x[(uint64_t)(n0 + r) * a.ldx + k0 + kk] : (int8_t)0;
        }
        __syncthreads();
#pragma unroll 4
        for (int w = 0; w < 16; ++w) {
            int32_t vw[4], vx[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                vw[i] = *reinterpret_cast<const int32_t *>(&tile_w[tm + 16 * i][4 * w]);
                vx[i] = *reinterpret_cast<const int32_t *>(&tile_x[tn + 16 * i][4 * w]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(vw[i], vx[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t channel = m0 + tm + 16 * i;
        if (channel >= a.m) continue;
        const float sw = a.sw[channel], bias = a.bias ? a.bias[channel] : 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t token = n0 + tn + 16 * j;
            if (token < a.n)
                i8_store(a.y, channel + (uint64_t)token * a.ldy, a.y_type, fmaf((float)acc[i][j] * a.sx[token], sw, bias));
        }
    }
}
