// Constants of the 8-bit kernels that the device code (text-included by the generator) and the host planner
// (sgemm_i8.cpp) have to agree on.  Preprocessor definitions only.
#ifndef SGEMM_I8_PARAMS_HPP
#define SGEMM_I8_PARAMS_HPP

// element type codes of the entry points (the generator's DataType numbers)
#define SGEMM_I8_FP32 0u
#define SGEMM_I8_FP16 1u
#define SGEMM_I8_BF16 2u

// ---- linear: k per stage (one 128-byte swizzle span of int8), rows of W per CTA
#define I8_BK 128
#define I8_BM 128
// CTA pairs: each CTA holds 128 rows of W and half of the tile's tokens
#define I8_PAIR_THREADS 384
#define I8_PAIR_SMEM(bn, stages) ((stages) * (I8_BM + (bn) / 2) * I8_BK + 1024 + 256)
#define I8_HALF_BN 128
#define I8_HALF_STAGES 8
// few-token kernels: tile 128 channels x TN tokens, one tile and one K range per CTA, the CTAs of a cluster share a tile
#define I8_FEW_THREADS 128
#define I8_FEW_SMEM(tn, stages) ((stages) * (I8_BM + (tn)) * I8_BK + 1024 + 256)
#define I8_FEW_STAGES_16 6
#define I8_FEW_STAGES_32 5
#define I8_FEW_STAGES_64 4
#define I8_FEW_STAGES_128 6
// largest K whose integer sum cannot leave 32 bits: K * 128 * 128 < 2^31
#define I8_MAX_K 131071u

// ---- fallback kernels for operands TMA cannot describe: square tiles
#define I8_SIMT_TILE 64
#define I8_SIMT_THREADS 256

// ---- weight gradient: 256 x 256 tile per CTA pair, tokens per stage
#define I8W_BK 64
#define I8W_STAGES 7          // stages of G, raw checkpoint and scales in flight
#define I8W_A_STAGES 3        // widened A tiles
#define I8W_THREADS 896
#define I8W_RING_BYTES (I8W_A_STAGES * 2 * 128 * I8W_BK + I8W_STAGES * (2 * 128 * I8W_BK + 128 * I8W_BK + 4 * I8W_BK))
#define I8W_SMEM (I8W_RING_BYTES + 1024 + 256)
#define I8W_LAUNCH_REGS 72    // what 896 threads leave per thread; the register hand-over below starts from it
#define I8W_CHAIN 8           // stages accumulated inside the tensor core before the sum moves to FP32 registers

// ---- row kernels: threads of a block (more when one row takes more)
#define I8_ROW_THREADS 256

// What a launch has to agree on with the kernel's code: the cubin carries these words, and sgemm_open compares them with the library's
// own, so that a cubin and a library compiled from different sources are refused instead of running with too little shared memory.
#define SGEMM_I8_LAYOUT                                                                                                        \
    {                                                                                                                          \
        I8_FEW_SMEM(16, I8_FEW_STAGES_16), I8_FEW_SMEM(32, I8_FEW_STAGES_32), I8_FEW_SMEM(64, I8_FEW_STAGES_64),               \
            I8_FEW_SMEM(128, I8_FEW_STAGES_128), I8W_SMEM, I8W_BK, I8W_THREADS, I8_BM, I8_BK, I8_FEW_THREADS, I8_SIMT_TILE,    \
            I8_PAIR_SMEM(I8_HALF_BN, I8_HALF_STAGES), I8_PAIR_THREADS,                                                         \
            I8_SIMT_THREADS, I8_ROW_THREADS, SGEMM_I8_ARGS_VERSION                                                         \
    }
#define SGEMM_I8_LAYOUT_WORDS 16
#define SGEMM_I8_ARGS_VERSION 2   // raised with every change of an argument structure

#endif
