// A matrix product with its bias, activation and residual (lily_linear, include/lily_layers.h):
//
//   out[t, n] = act(sa[t] * sw[n] * sum_k a[t, k] * w[n, k] + bias[n]) + residual[t, n]
//
// The multiplier's M side takes the weights (128 outputs a tile) and its N side the tokens, so
// that few tokens waste nothing: a step's time is its weights' stream. A lane of tensor memory is
// then an output and a column a token: an epilogue thread owns one output (its scale and bias are two
// registers), and a warp writes 32 neighbouring outputs of a token at a time.
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>
#include <cstring>
#include <type_traits>

#include "../../include/lily_layers.h"
#include "handle.cuh"
#include "lmhead_args.cuh"
#include "tc.cuh"

namespace {

using namespace lily_host;
using namespace lily_tc;

constexpr uint32_t TILE_M = 128;       // outputs of a tile
constexpr uint32_t BLOCK_BYTES = 128;  // of a row's columns, a step of the pipeline: 64 bf16, 128 e4m3
constexpr uint32_t A_STAGE = TILE_M * BLOCK_BYTES;
constexpr uint32_t FULL = 0xFFFFFFFFu;

struct LinearArgs {
    CUtensorMap w_map;  // [outputs, columns], boxes of a tile's rows (many tokens: a block's 128) x 128 bytes, 128-byte swizzle
    CUtensorMap a_map;  // [tokens, columns], boxes of a token tile (many tokens: half of one) x 128 bytes
    CUtensorMap out_map, residual_map;  // many tokens, `copies`: bf16 [tokens, outputs], boxes of half a tile x 32 outputs
    const float *a_scales, *w_scales;
    const void *bias, *residual;
    void *out;
    uint64_t residual_ld, out_ld;
    uint32_t tokens, outputs;
    uint32_t blocks;        // steps of BLOCK_BYTES in a row
    uint32_t tile_outputs;  // few tokens: of a tile, a multiple of 8
    uint32_t token_tiles;   // many tokens
    uint32_t tile_tokens;   // many tokens: of a tile, a multiple of 32
    uint32_t copies;        // many tokens: out and residual go through shared memory
    uint32_t shares;        // many tokens: pairs of a cluster that share a tile's columns
    uint32_t stages;        // of the pipeline
    uint32_t out_f32, bias_f32, activation;
    uint32_t *status_word;
    uint64_t wait_ns;
    uint32_t lost_stage;    // test hook: the first block leaves out the copies of this step (~0: none)
};

// The normal distribution's integral up to v, (1 + erf(v / sqrt(2))) / 2. Of |v| on the far side it is exp(-v^2 / 2) t p(t)
// with t = 1 / (1 + 0.36 |v|), and p a polynomial: minimax fits (weighted least squares on 0..14, the weights driven
// to an even error) of the relative error, so that the far side keeps its digits, where 1 + erf cancels. For results in
// 32 bits p is 2^-23.9 off, its evaluation 2^-21 up to |v| = 3, and beyond as much as v, rounded, moves the function (its
// square loses v^2 2^-24); for results of 8 bits, whose half step is 2^-8, two terms fewer and 2^-20.1. No lane takes a
// branch alone. (8192 x 512 x 8192, GELU: bf16 outs 116..127 us, f32 152..158; erfcf took 219 for f32.)
template <bool SHORT_OUT>
__device__ __forceinline__ float normal_integral(float v) {
    float t, e;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(0.36f, fabsf(v), 1.0f)));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v * v * -0.72134752f));  // (log2(e) / 2)
    float p;
    if (SHORT_OUT) {
        p = fmaf(0.0470560603f, t, -0.179763928f);
        p = fmaf(p, t, 0.180952996f);
        p = fmaf(p, t, 0.0265499875f);
        p = fmaf(p, t, 0.139719039f);
        p = fmaf(p, t, 0.141772494f);
        p = fmaf(p, t, 0.143713042f);
    } else {
        p = fmaf(-0.0296530277f, t, 0.136437729f);
        p = fmaf(p, t, -0.216858417f);
        p = fmaf(p, t, 0.0993036404f);
        p = fmaf(p, t, 0.00534496736f);
        p = fmaf(p, t, 0.0935714766f);
        p = fmaf(p, t, 0.124633908f);
        p = fmaf(p, t, 0.14359735f);
        p = fmaf(p, t, 0.143622339f);
    }
    const float tail = p * t * e;
    return v < 0.0f ? tail : 1.0f - tail;
}

// C values through the activation. One branch for all of them: with the branch inside, sixteen
// copies of every function's code lay in the epilogue's loop, which then ran from instruction misses
// (4099 x 4096 x 4096 without an activation 120 us, with a residual 331).
template <uint32_t C>
__device__ __forceinline__ void activate(float (&v)[C], uint32_t activation, bool short_out) {
    if (activation == LILY_ACT_NONE) {
    } else if (activation == LILY_ACT_RELU) {
#pragma unroll
        for (uint32_t j = 0; j < C; ++j) {
            v[j] = v[j] < 0.0f ? 0.0f : v[j];  // (a NaN stays)
        }
    } else if (activation == LILY_ACT_SILU) {
#pragma unroll
        for (uint32_t j = 0; j < C; ++j) {
            v[j] = __fdividef(v[j], 1.0f + expf(-v[j]));
        }
    } else if (activation == LILY_ACT_GELU && short_out) {
#pragma unroll
        for (uint32_t j = 0; j < C; ++j) {
            v[j] *= normal_integral<true>(v[j]);
        }
    } else if (activation == LILY_ACT_GELU) {
#pragma unroll
        for (uint32_t j = 0; j < C; ++j) {
            v[j] *= normal_integral<false>(v[j]);
        }
    } else {
#pragma unroll
        for (uint32_t j = 0; j < C; ++j) {
            const float u = 0.79788456f * (v[j] + 0.044715f * v[j] * v[j] * v[j]);
            v[j] = __fdividef(v[j], 1.0f + expf(-2.0f * u));  // (1 + tanh(u)) / 2 = 1 / (1 + exp(-2 u))
        }
    }
}

// What a thread of the epilogue knows of its output n.
struct Output {
    float scale, bias;
    bool live;
};

__device__ __forceinline__ Output output_of(const LinearArgs &a, uint32_t n) {
    Output o = {1.0f, 0.0f, n < a.outputs};
    if (o.live && a.w_scales != nullptr) {
        o.scale = __ldg(a.w_scales + n);
    }
    if (o.live && a.bias != nullptr) {
        o.bias = a.bias_f32 ? __ldg(static_cast<const float *>(a.bias) + n)
                            : __bfloat162float(static_cast<const __nv_bfloat16 *>(a.bias)[n]);
    }
    return o;
}

// The residuals of output n and of up to C tokens from t on.
template <uint32_t C>
__device__ __forceinline__ void residuals_of(const LinearArgs &a, const Output &o, uint32_t t, uint32_t n, uint32_t live,
                                             float (&r)[C]) {
    if (a.residual == nullptr || !o.live) {
#pragma unroll
        for (uint32_t j = 0; j < C; ++j) {
            r[j] = 0.0f;
        }
    } else if (a.out_f32) {
        const float *p = static_cast<const float *>(a.residual) + (uint64_t)t * a.residual_ld + n;
#pragma unroll
        for (uint32_t j = 0; j < C; ++j) {
            r[j] = j < live ? p[j * a.residual_ld] : 0.0f;
        }
    } else {
        const __nv_bfloat16 *p = static_cast<const __nv_bfloat16 *>(a.residual) + (uint64_t)t * a.residual_ld + n;
#pragma unroll
        for (uint32_t j = 0; j < C; ++j) {
            r[j] = j < live ? __bfloat162float(p[j * a.residual_ld]) : 0.0f;
        }
    }
}

// The scales of up to 128 tokens from t on, token 32 i + j's with lane j: asked for before the sums are there.
struct TokenScales {
    float v[4];

    __device__ __forceinline__ TokenScales(const LinearArgs &a, uint32_t t, uint32_t live) {
        const uint32_t lane = threadIdx.x % 32u;
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            v[i] = a.a_scales != nullptr && 32u * i + lane < live ? __ldg(a.a_scales + t + 32u * i + lane) : 0.0f;
        }
    }

    __device__ __forceinline__ float of(uint32_t c) const { return c < 64u ? (c < 32u ? v[0] : v[1]) : c < 96u ? v[2] : v[3]; }
};

// The sums v of an output and of C tokens from the c-th of `s` on (all of them among the same 32), finished; and
// written, up to `live` of them. (A whole warp.)
template <uint32_t C>
__device__ __forceinline__ void finish_sums(const LinearArgs &a, const Output &o, const TokenScales &s, uint32_t c, float (&v)[C],
                                            const float (&r)[C]) {
    if (a.a_scales != nullptr) {
        const float mine = s.of(c);
#pragma unroll
        for (uint32_t j = 0; j < C; ++j) {
            v[j] *= __shfl_sync(FULL, mine, c % 32u + j) * o.scale;
        }
    }
#pragma unroll
    for (uint32_t j = 0; j < C; ++j) {
        v[j] += o.bias;
    }
    activate(v, a.activation, !a.out_f32);
#pragma unroll
    for (uint32_t j = 0; j < C; ++j) {
        v[j] += r[j];
    }
}

template <uint32_t C>
__device__ __forceinline__ void finish(const LinearArgs &a, const Output &o, const TokenScales &s, uint32_t c, uint32_t t, uint32_t n,
                                       uint32_t live, float (&v)[C], const float (&r)[C]) {
    finish_sums(a, o, s, c, v, r);
    if (!o.live) {
    } else if (a.out_f32) {
        float *p = static_cast<float *>(a.out) + (uint64_t)t * a.out_ld + n;
#pragma unroll
        for (uint32_t j = 0; j < C; ++j) {
            if (j < live) {
                p[j * a.out_ld] = v[j];
            }
        }
    } else {
        __nv_bfloat16 *p = static_cast<__nv_bfloat16 *>(a.out) + (uint64_t)t * a.out_ld + n;
#pragma unroll
        for (uint32_t j = 0; j < C; ++j) {
            if (j < live) {
                p[j * a.out_ld] = __float2bfloat16_rn(v[j]);
            }
        }
    }
}

// D binary32; A and B both bf16 (kind::f16) or both e4m3 (kind::f8f6f4), both K-major.
template <bool E4M3>
__device__ __forceinline__ uint32_t product_desc(uint32_t m, uint32_t n) {
    return (1u << 4) | (E4M3 ? 0u : (1u << 7) | (1u << 10)) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

// D[tmem] (+)= A[smem] * B[smem]^T over 32 bytes of columns.
template <bool E4M3>
__device__ __forceinline__ void mma_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    if (E4M3) {
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
            ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
            : "memory");
    } else {
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
            ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
            : "memory");
    }
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

__device__ __forceinline__ uint32_t at_rank(uint32_t addr, uint32_t rank) {
    uint32_t there;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(addr), "r"(rank));
    return there;
}

// ------------------------------------------------------------------ few tokens --
//
// Up to 32 tokens, of bf16 heads up to 64. Many tiles, of up to 128 outputs x N tokens: a block has one after the other, and finishes one
// while it multiplies the next; the tile's outputs are as many as give all blocks the same (1 x 4096 x 40000: with
// 128 for 313 tiles on 296 blocks 60 us, with 72 51: 6.4 TB/s). Few: a cluster has one of 128, whose columns its blocks share out evenly. Each
// sums its share in tensor memory, then sends every token's column of sums to the block that finishes that
// token, which adds the shares up in the blocks' order.
//
// What bounds it: the weights' stream (16 x 2048 x 151936 94 us, 6.7 TB/s); below about 50 MB of them a launch's
// fixed costs, 3 us, and a copy's way of a microsecond for as many steps as a block has stages.
//
// A block's warps: 0 asks for the copies, 1 issues the multiplies, 2 to 5 are the epilogue.
template <uint32_t N>
struct Few {
    static constexpr uint32_t THREADS = 192;
    static constexpr uint32_t B_STAGE = N * BLOCK_BYTES;
    static constexpr uint32_t PART_BYTES = N * TILE_M * 4u;
    // Two blocks on an SM.
    static constexpr uint32_t MOST_STAGES = 10;
    static constexpr uint32_t RING = (N == 16u ? 5u : 4u) * (A_STAGE + B_STAGE);  // bytes of stages
    // The sums that blocks send one another have a place of their own: a block may send as soon as the other runs.
    // (64 tokens come here with tiles for all blocks.)
    static constexpr bool SHARES = N <= 32u;
    // Sums of successive steps go into accumulators in turn: shorter chains of additions. Two sets of them: a
    // tile is finished while the block's next one is multiplied.
    static constexpr uint32_t ACCS = 2, SETS = 2;
    static constexpr uint32_t COLS = SETS * ACCS * N;
    static constexpr uint32_t PART = RING;
    static constexpr uint32_t BARS = RING + (SHARES ? PART_BYTES : 0u);
    static constexpr uint32_t EMPTY = BARS + 8u * MOST_STAGES;
    static constexpr uint32_t ACC_FULL = EMPTY + 8u * MOST_STAGES;
    static constexpr uint32_t ACC_EMPTY = ACC_FULL + 8u * SETS;
    static constexpr uint32_t FINAL = ACC_EMPTY + 8u * SETS;
    static constexpr uint32_t TMEM_ADDR = FINAL + 8u;
    static constexpr uint32_t ABORT = TMEM_ADDR + 4u;
    static constexpr uint32_t BYTES = ABORT + 4u + 1024u;
    static_assert(BYTES <= 227u * 1024u && BYTES > 76u * 1024u, "at most two blocks on an SM");
    // (A multiply reads 128 rows of every stage, the last one's too: they lie in the ring.)
    static constexpr uint32_t stages_of(uint32_t outputs) {
        const uint32_t stage = outputs * BLOCK_BYTES + B_STAGE, n = (RING - A_STAGE) / stage + 1u, all = RING / stage;
        return n < all ? (n < MOST_STAGES ? n : MOST_STAGES) : all < MOST_STAGES ? all : MOST_STAGES;
    }
    static_assert(COLS >= 32u && COLS <= 256u && (COLS & (COLS - 1u)) == 0u, "tensor memory of two blocks on an SM");
};

template <uint32_t N, bool E4M3>
__global__ void __launch_bounds__(192) linear_few_kernel(const __grid_constant__ LinearArgs a) {
    using S = Few<N>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *smem = smem_raw + (base - smem_u32(smem_raw));
    volatile uint32_t *abort_word = reinterpret_cast<volatile uint32_t *>(smem + S::ABORT);
    const uint32_t tid = threadIdx.x, warp = __shfl_sync(FULL, tid / 32u, 0), lane = tid % 32u;
    uint32_t rank, shares;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(shares));
    const uint32_t tile0 = blockIdx.x / shares, stride = gridDim.x / shares;
    const uint32_t tiles = (a.outputs + a.tile_outputs - 1u) / a.tile_outputs;
    const uint32_t stages = a.stages, a_stage = a.tile_outputs * BLOCK_BYTES, stage = a_stage + S::B_STAGE;
    const auto output_tile = [&](uint32_t tile) { return tile * a.tile_outputs; };
    const uint32_t block0 = (uint32_t)((uint64_t)a.blocks * rank / shares);
    const uint32_t steps = (uint32_t)((uint64_t)a.blocks * (rank + 1u) / shares) - block0;

    if (tid == 0) {
        for (uint32_t s = 0; s < S::MOST_STAGES; ++s) {
            mbar_init(base + S::BARS + 8 * s, 1);
            mbar_init(base + S::EMPTY + 8 * s, 1);
        }
        for (uint32_t b = 0; b < S::SETS; ++b) {
            mbar_init(base + S::ACC_FULL + 8 * b, 1);
            mbar_init(base + S::ACC_EMPTY + 8 * b, 4);
        }
        mbar_init(base + S::FINAL, 1);
        *abort_word = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1u) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base + S::TMEM_ADDR),
                     "r"(S::COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(smem + S::TMEM_ADDR);
    if (S::SHARES && shares > 1u) {
        cluster_arrive();  // (this block has begun: the others may write into its shared memory)
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // (Behind the allocation: a block of the next launch that held tensor memory before all of this
    // launch's have theirs would wait for them, and they for it.)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    if (warp == 0u) {
        if (lane == 0u) {
            uint32_t asked = 0, parity = 0, i = 0, s = 0, use = 0;
            for (uint32_t tile = tile0; tile < tiles; tile += stride) {
                const int32_t output0 = (int32_t)output_tile(tile);
                for (uint32_t k = 0; k < steps; ++k, ++i) {
                    if (mbar_wait(base + S::EMPTY + 8 * s, use ^ 1u, abort_word, a.wait_ns)) {
                        tile = tiles - stride;  // (the last one)
                        break;
                    }
                    const uint32_t at = s, bar = base + S::BARS + 8 * s, to = base + s * stage, phase = use;
                    s = s + 1u == stages ? 0u : s + 1u;
                    use ^= s == 0u;
                    const int32_t x = (int32_t)((block0 + k) * (E4M3 ? BLOCK_BYTES : BLOCK_BYTES / 2u));
                    if (i == a.lost_stage && blockIdx.x == 0u) {
                        continue;  // (test hook: the stage never fills)
                    }
                    asked |= 1u << at;
                    parity = (parity & ~(1u << at)) | phase << at;
                    mbar_expect_tx(bar, stage);
                    tma_load_2d(to, &a.w_map, bar, x, output0);
                    tma_load_2d(to + a_stage, &a.a_map, bar, x, 0);
                }
            }
            if (*abort_word) {  // the copies asked for land in this block's shared memory: it stays until they have
                for (s = 0; s < stages; ++s) {
                    if (asked >> s & 1u) {
                        mbar_drain(base + S::BARS + 8 * s, parity >> s & 1u, a.wait_ns);
                    }
                }
            }
        }
        __syncwarp();
    } else if (warp == 1u) {
        const bool leader = elect_one();
        const uint32_t idesc = product_desc<E4M3>(TILE_M, N);
        uint32_t s = 0, use = 0, turn = 0;
        bool gave_up = false;
        for (uint32_t tile = tile0; tile < tiles && !gave_up; tile += stride, ++turn) {
            const uint32_t b = turn % S::SETS;
            if (warp_wait(base + S::ACC_EMPTY + 8 * b, (turn / S::SETS & 1u) ^ 1u, abort_word, a.wait_ns)) {
                break;
            }
            for (uint32_t k = 0; k < steps; ++k) {
                if (warp_wait(base + S::BARS + 8 * s, use, abort_word, a.wait_ns)) {
                    gave_up = true;
                    break;
                }
                tc_fence_after();
                if (leader) {
                    const uint64_t adesc = operand_desc(base + s * stage), bdesc = operand_desc(base + s * stage + a_stage);
#pragma unroll
                    for (uint32_t q = 0; q < 4u; ++q) {
                        mma_ss<E4M3>(tmem + (b * S::ACCS + k % S::ACCS) * N, adesc + 2u * q, bdesc + 2u * q, idesc, k >= S::ACCS || q > 0u);
                    }
                    mma_commit(base + S::EMPTY + 8 * s);
                }
                __syncwarp();
                s = s + 1u == stages ? 0u : s + 1u;
                use ^= s == 0u;
            }
            if (leader && !gave_up) {
                mma_commit(base + S::ACC_FULL + 8 * b);
            }
            __syncwarp();
        }
        if (leader) {
            mma_commit(base + S::FINAL);
            mbar_drain(base + S::FINAL, 0u, a.wait_ns);  // (nothing is freed under a multiply, on any way out)
        }
        __syncwarp();
    }

    const uint32_t quad = warp % 4u, row = quad * 32u + lane;  // the epilogue's lanes of tensor memory
    const uint32_t accs = min(S::ACCS, steps), from = tmem + (quad * 32u << 16);
    // Sixteen tokens' sums of this thread's output, of set b.
    const auto sums_of = [&](uint32_t b, uint32_t c, float (&v)[16]) {
        uint32_t q[S::ACCS][16];
#pragma unroll
        for (uint32_t k = 0; k < S::ACCS; ++k) {
            if (k < accs) {
                tmem_ld16(from + (b * S::ACCS + k) * N + c, q[k]);
            }
        }
        tmem_ld_wait();
#pragma unroll
        for (uint32_t j = 0; j < 16u; ++j) {
            v[j] = __uint_as_float(q[0][j]);
        }
#pragma unroll
        for (uint32_t k = 1; k < S::ACCS; ++k) {
            if (k < accs) {
#pragma unroll
                for (uint32_t j = 0; j < 16u; ++j) {
                    v[j] += __uint_as_float(q[k][j]);
                }
            }
        }
    };
    if (!S::SHARES || shares == 1u) {
        uint32_t turn = 0;
        for (uint32_t tile = tile0; warp >= 2u && tile < tiles; tile += stride, ++turn) {
            const uint32_t b = turn % S::SETS, n = output_tile(tile) + row, live = a.tokens;
            Output o = output_of(a, n);
            o.live = o.live && row < a.tile_outputs;  // (the other rows multiply what lies in the stage)
            const TokenScales scales(a, 0u, live);
            float r[16];
            residuals_of(a, o, 0u, n, live, r);  // (asked for a round ahead, here and below)
            if (warp_wait(base + S::ACC_FULL + 8 * b, turn / S::SETS & 1u, abort_word, a.wait_ns)) {
                break;
            }
            tc_fence_after();
            for (uint32_t c = 0; c < live; c += 16u) {
                float v[16], next[16];
                residuals_of(a, o, c + 16u, n, live > c + 16u ? live - c - 16u : 0u, next);
                sums_of(b, c, v);
                if (c + 16u >= live) {  // (the sums are in registers)
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0u) {
                        mbar_arrive(base + S::ACC_EMPTY + 8 * b);
                    }
                }
                finish(a, o, scales, c, c, n, live - c, v, r);
#pragma unroll
                for (uint32_t j = 0; j < 16u; ++j) {
                    r[j] = next[j];
                }
            }
        }
    } else {
        // Token c is finished by block c / per; its sums lie there at [share][output][c % per], four tokens
        // (or both) side by side, which an output's thread sends and takes together. (One by one the
        // sums of 128 tokens took 3.6 us to send and 13 to add up; the pairs have those now.)
        const uint32_t n = output_tile(tile0) + row, live = a.tokens;
        const uint32_t per = N / shares, log_per = 31u - __clz(per);  // (powers of two)
        const uint32_t first = rank * per, mine = first < live ? min(per, live - first) : 0u;
        const uint32_t quads = per / 4u;
        const auto part_at = [&](uint32_t share, uint32_t c) {  // (neighbours' quads lie in different banks)
            return base + S::PART + (share * TILE_M + row) * per * 4u + (((c / 4u) ^ (row & (quads - 1u))) * 16u);
        };
        // What does not depend on the sums is asked for before they are there.
        Output o = {1.0f, 0.0f, false};
        const TokenScales scales(a, first, warp >= 2u ? mine : 0u);
        float r[16];
        if (warp >= 2u) {
            o = output_of(a, n);
            residuals_of(a, o, first, n, mine, r);
        }
        if (warp >= 2u) {
            warp_wait(base + S::ACC_FULL, 0u, abort_word, a.wait_ns);
            tc_fence_after();
        }
        __syncwarp();
        cluster_wait();
        if (warp >= 2u) {
            for (uint32_t c = 0; c < live; c += 16u) {
                float v[16];
                sums_of(0u, c, v);
                if (per == 2u) {
#pragma unroll
                    for (uint32_t j = 0; j < 16u; j += 2u) {
                        if (c + j < live) {
                            const uint32_t there = at_rank(base + S::PART + (rank * TILE_M + row) * 8u, (c + j) / 2u);
                            asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(there), "f"(v[j]), "f"(v[j + 1u]) : "memory");
                        }
                    }
                } else {
#pragma unroll
                    for (uint32_t j = 0; j < 16u; j += 4u) {
                        if (c + j < live) {
                            const uint32_t there = at_rank(part_at(rank, (c + j) & (per - 1u)), (c + j) >> log_per);
                            asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(there), "f"(v[j]), "f"(v[j + 1u]),
                                         "f"(v[j + 2u]), "f"(v[j + 3u])
                                         : "memory");
                        }
                    }
                }
            }
        }
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        if (warp >= 2u) {
            if (per == 2u) {
                float v[2] = {0.0f, 0.0f}, r2[2] = {r[0], r[1]};
                const float2 *part = reinterpret_cast<const float2 *>(smem + S::PART) + row;
#pragma unroll
                for (uint32_t k = 0; k < 8u; ++k) {  // (two tokens a block: eight blocks)
                    const float2 p = part[k * TILE_M];
                    v[0] += p.x, v[1] += p.y;
                }
                if (mine > 0u) {
                    finish(a, o, scales, 0u, first, n, mine, v, r2);
                }
            } else {
                const auto finish_all = [&](auto at_once) {
                    constexpr uint32_t C = decltype(at_once)::value;
                    for (uint32_t c = 0; c < mine; c += C) {
                        float v[C] = {}, rc[C];
                        if (c == 0u) {
#pragma unroll
                            for (uint32_t j = 0; j < C; ++j) {
                                rc[j] = r[j];
                            }
                        } else {
                            residuals_of(a, o, first + c, n, mine - c, rc);
                        }
                        for (uint32_t k = 0; k < shares; ++k) {
#pragma unroll
                            for (uint32_t j = 0; j < C; j += 4u) {
                                const float4 p = *reinterpret_cast<const float4 *>(smem + (part_at(k, c + j) - base));
                                v[j] += p.x, v[j + 1u] += p.y, v[j + 2u] += p.z, v[j + 3u] += p.w;
                            }
                        }
                        finish(a, o, scales, c, first + c, n, mine - c, v, rc);
                    }
                };
                if (per == 4u) {  // (no code for tokens that are not there: most of it runs once, and waits for itself)
                    finish_all(std::integral_constant<uint32_t, 4>());
                } else if (per == 8u) {
                    finish_all(std::integral_constant<uint32_t, 8>());
                } else {
                    finish_all(std::integral_constant<uint32_t, 16>());
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (*abort_word) {
        stay_for_landings();
    }
    tc_fence_after();
    if (warp == 1u) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::COLS) : "memory");
    }
    if (tid == 0 && *abort_word) {
        atomicOr(a.status_word, 1u << lily_head::STATUS_TIMEOUT_BIT);
    }
}

// ----------------------------------------------------------------- many tokens --
//
// From 33 tokens on, of bf16 heads from 65. Tiles of 256 outputs x up to 256 tokens, each by a pair of blocks (a cluster of two on neighbouring
// SMs) whose tensor cores multiply together: either block holds 128 outputs' weights and half of the tokens in
// shared memory, and the pair's multiply reads both. That halves the bytes that a multiply takes
// out of each SM's shared memory, which one block alone is bound by. The pairs stay for all of the launch; an
// accumulator is finished (scale, bias, activation, residual) while the next tile is multiplied
// into the other one. bf16 outs and residuals go through shared memory where their rows allow it: the
// residuals come while the tile is multiplied, and nothing in the epilogue waits for global memory. (Read
// and written in place, 64 bytes a warp at a time, they took 55 us of the 153 of 4099 x 4096 x 4096.)
//
// Where the tiles are few, two or four pairs of a cluster share the columns of one (256 x 8192 x 1024: 35 us
// alone, 15 by four pairs). The stages are as many as fit beside the rest: few tokens make small ones.
//
// What bounds it: at 8192 x 4096 x 8192 (bf16 375 to 400 us, 1.4 PFLOP/s; e4m3 216 us, 2.5) and 4099 x 4096 x 4096
// (96 to 104 us) the tiles that all SMs together take out of L2, 11 TB/s, and with the tensor cores
// busy for three quarters of the time, the board's power; below about 1000 tokens the launch, the pipeline's
// first copies and the last tile's end, 5 us together.
//
// A block's warps: 0 and 10 ask for the block's copies in turn (one alone took 0.25 us for a step's two: 300 x 8192 x 2048
// 23.8 us, with two warps 20.4; three and four give the same), 1 issues the pair's multiplies (in the first block
// of the pair alone), 2 to 9 are the epilogue, two for each quarter of tensor memory's lanes.
struct Many {
    static constexpr uint32_t ASKERS = 2;
    static constexpr uint32_t THREADS = 288 + 32 * ASKERS;
    static constexpr uint32_t TILE = 256;          // of outputs, and the most of tokens
    static constexpr uint32_t MOST_STAGES = 11;
    static constexpr uint32_t RING = 5u * 2u * A_STAGE;  // bytes of stages: a block's half of the weights, and of the tokens
    static constexpr uint32_t WARP_TILE = 128u * 64u;  // bf16 outs of a warp of the epilogue: 128 tokens, 32 outputs
    static constexpr uint32_t ACCS = 2;
    static constexpr uint32_t EPI_WARPS = 8;
    static constexpr uint32_t ASKER = 2u + EPI_WARPS;  // the second warp that asks for copies
    static constexpr uint32_t COLS = ACCS * TILE;
    static constexpr uint32_t OUT = RING;          // (without outs and residuals in shared memory: stages, too)
    static constexpr uint32_t FULL_BARS = OUT + EPI_WARPS * WARP_TILE;  // in the first block: both blocks' copies are there
    static constexpr uint32_t EMPTY = FULL_BARS + 8u * MOST_STAGES;
    static constexpr uint32_t ACC_FULL = EMPTY + 8u * MOST_STAGES;
    static constexpr uint32_t ACC_EMPTY = ACC_FULL + 8u * ACCS;     // in the first block: both blocks have read it
    static constexpr uint32_t FINAL = ACC_EMPTY + 8u * ACCS;
    static constexpr uint32_t RESIDUAL = FINAL + 8u;                // [EPI_WARPS] the warp's residuals are there
    static constexpr uint32_t TMEM_ADDR = RESIDUAL + 8u * EPI_WARPS;
    static constexpr uint32_t ABORT = TMEM_ADDR + 4u;
    static constexpr uint32_t BYTES = ABORT + 4u + 1024u;
    static_assert(BYTES <= 227u * 1024u, "shared memory of one block");

    static constexpr uint32_t stage_bytes(uint32_t tokens) { return A_STAGE + tokens / 2u * BLOCK_BYTES; }
    static constexpr uint32_t stages_of(uint32_t tokens, bool copies) {
        const uint32_t n = (copies ? RING : FULL_BARS) / stage_bytes(tokens);
        return n < MOST_STAGES ? n : MOST_STAGES;
    }
};

// A copy into this block's shared memory whose bytes complete a barrier of either block of the pair.
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap *map, uint32_t cluster_bar, int32_t x, int32_t y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(cluster_bar), "r"(x), "r"(y)
        : "memory");
}

// A tile out of shared memory; parts beyond the tensor are left out.
__device__ __forceinline__ void tma_store_2d(const CUtensorMap *map, uint32_t src, int32_t x, int32_t y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];"
                 ::"l"(reinterpret_cast<uint64_t>(map)), "r"(src), "r"(x), "r"(y)
                 : "memory");
}

template <bool E4M3>
__device__ __forceinline__ void mma_ss_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    if (E4M3) {
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
            ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
            : "memory");
    } else {
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
            ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
            : "memory");
    }
}

// Arrives at this barrier of both blocks of the pair, whose first in the cluster is `first`, once the multiplies
// issued so far have run.
__device__ __forceinline__ void mma_commit_pair(uint32_t bar, uint32_t first) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"((uint16_t)(3u << first))
        : "memory");
}

template <bool E4M3>
__global__ void __launch_bounds__(Many::THREADS, 1) linear_many_kernel(const __grid_constant__ LinearArgs a) {
    using S = Many;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *smem = smem_raw + (base - smem_u32(smem_raw));
    volatile uint32_t *abort_word = reinterpret_cast<volatile uint32_t *>(smem + S::ABORT);
    const uint32_t tid = threadIdx.x, warp = __shfl_sync(FULL, tid / 32u, 0), lane = tid % 32u;
    const bool epilogue = warp >= 2u && warp < S::ASKER;
    uint32_t in_cluster;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(in_cluster));
    const uint32_t rank = in_cluster & 1u, first = in_cluster & ~1u, share = in_cluster / 2u;
    const uint32_t pair = blockIdx.x / (2u * a.shares), pairs = gridDim.x / (2u * a.shares);  // (clusters, with shares)
    const uint32_t stages = a.stages, stage = A_STAGE + a.tile_tokens / 2u * BLOCK_BYTES;
    const uint32_t from_step = share * a.blocks / a.shares, to_step = (share + 1u) * a.blocks / a.shares;
    const uint32_t output_tiles = (a.outputs + S::TILE - 1u) / S::TILE, tiles = output_tiles * a.token_tiles;

    if (tid == 0) {
        for (uint32_t s = 0; s < S::MOST_STAGES; ++s) {
            mbar_init(base + S::FULL_BARS + 8 * s, 1);
            mbar_init(base + S::EMPTY + 8 * s, 1);
        }
        for (uint32_t b = 0; b < S::ACCS; ++b) {
            mbar_init(base + S::ACC_FULL + 8 * b, 1);
            mbar_init(base + S::ACC_EMPTY + 8 * b, 2u * S::EPI_WARPS);
        }
        mbar_init(base + S::FINAL, 1);
        for (uint32_t w = 0; w < S::EPI_WARPS; ++w) {
            mbar_init(base + S::RESIDUAL + 8 * w, 1);
        }
        *abort_word = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1u) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base + S::TMEM_ADDR),
                     "r"(S::COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_arrive();
    cluster_wait();  // (both blocks' barriers and tensor memory are there)
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(smem + S::TMEM_ADDR);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // (behind the allocation, as above)

    if (warp == 0u || warp >= S::ASKER) {
        if (lane == 0u) {
            const uint32_t which = warp == 0u ? 0u : warp - S::ASKER + 1u;
            uint32_t i = 0, s = which, phase = 0;  // steps so far; of the ring
            bool gave_up = false;
            for (uint32_t tile = pair; tile < tiles && !gave_up; tile += pairs) {
                const int32_t output0 = (int32_t)(tile / a.token_tiles * S::TILE + rank * TILE_M);
                const int32_t token0 = (int32_t)(tile % a.token_tiles * a.tile_tokens + rank * (a.tile_tokens / 2u));
                for (uint32_t k = from_step; k < to_step; ++k, ++i) {
                    if (i % S::ASKERS != which) {
                        continue;
                    }
                    if (mbar_wait(base + S::EMPTY + 8 * s, phase ^ 1u, abort_word, a.wait_ns)) {
                        gave_up = true;
                        break;
                    }
                    const uint32_t bar = base + S::FULL_BARS + 8 * s, to = base + s * stage;
                    s += S::ASKERS;
                    if (s >= stages) {
                        s -= stages;
                        phase ^= 1u;
                    }
                    const int32_t x = (int32_t)(k * (E4M3 ? BLOCK_BYTES : BLOCK_BYTES / 2u));
                    if (i == a.lost_stage && blockIdx.x == 0u) {
                        continue;  // (test hook: the stage never fills)
                    }
                    if (rank == 0u) {
                        mbar_expect_tx(bar, 2u * A_STAGE + a.tile_tokens * BLOCK_BYTES);
                    }
                    tma_load_2d_pair(to, &a.w_map, at_rank(bar, first), x, output0);
                    tma_load_2d_pair(to + A_STAGE, &a.a_map, at_rank(bar, first), x, token0);
                }
            }
        }
        __syncwarp();
    } else if (warp == 1u && rank == 0u) {
        const bool leader = elect_one();
        const uint32_t idesc = product_desc<E4M3>(2u * TILE_M, a.tile_tokens);
        uint32_t s = 0, phase = 0, turn = 0;
        bool gave_up = false;
        for (uint32_t tile = pair; tile < tiles && !gave_up; tile += pairs, ++turn) {
            const uint32_t b = turn % S::ACCS;
            if (warp_wait(base + S::ACC_EMPTY + 8 * b, (turn / S::ACCS & 1u) ^ 1u, abort_word, a.wait_ns)) {
                break;
            }
            for (uint32_t k = from_step; k < to_step; ++k) {
                if (warp_wait(base + S::FULL_BARS + 8 * s, phase, abort_word, a.wait_ns)) {
                    gave_up = true;
                    break;
                }
                tc_fence_after();
                if (leader) {
                    const uint64_t adesc = operand_desc(base + s * stage), bdesc = operand_desc(base + s * stage + A_STAGE);
#pragma unroll
                    for (uint32_t q = 0; q < 4u; ++q) {
                        mma_ss_pair<E4M3>(tmem + b * S::TILE, adesc + 2u * q, bdesc + 2u * q, idesc, k > from_step || q > 0u);
                    }
                    mma_commit_pair(base + S::EMPTY + 8 * s, first);
                }
                __syncwarp();
                s = s + 1u == stages ? 0u : s + 1u;
                phase ^= s == 0u;
            }
            if (leader && !gave_up) {
                mma_commit_pair(base + S::ACC_FULL + 8 * b, first);
            }
            __syncwarp();
        }
        if (leader) {
            mma_commit_pair(base + S::FINAL, first);
            mbar_drain(base + S::FINAL, 0u, a.wait_ns);  // (nothing is freed under a multiply, on any way out)
        }
        __syncwarp();
    } else if (epilogue && a.shares == 1u) {
        const uint32_t quad = warp % 4u, half = (warp - 2u) / 4u;
        uint32_t turn = 0, loaded = 0;  // tiles; residuals asked for
        for (uint32_t tile = pair; tile < tiles; tile += pairs, ++turn) {
            const uint32_t b = turn % S::ACCS;
            const uint32_t n = tile / a.token_tiles * S::TILE + rank * TILE_M + quad * 32u + lane;
            const uint32_t tokens = a.tile_tokens / 2u, token0 = tile % a.token_tiles * a.tile_tokens + half * tokens;
            const uint32_t live = token0 < a.tokens ? min(tokens, a.tokens - token0) : 0u;
            const uint32_t from = tmem + (quad * 32u << 16) + b * S::TILE + half * tokens;
            const Output o = output_of(a, n);
            const TokenScales scales(a, token0, live);
            if (a.copies) {
                const uint32_t w = warp - 2u, mine = base + S::OUT + w * S::WARP_TILE + lane * 2u, bar = base + S::RESIDUAL + 8 * w;
                const bool any = live > 0u && n - lane < a.outputs;
                if (any && lane == 0u) {
                    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // (the last tile's outs have left)
                    if (a.residual != nullptr) {
                        mbar_expect_tx(bar, tokens * 64u);
                        tma_load_2d(mine, &a.residual_map, bar, (int32_t)n, (int32_t)token0);
                        ++loaded;
                    }
                }
                __syncwarp();
                if (warp_wait(base + S::ACC_FULL + 8 * b, turn / S::ACCS & 1u, abort_word, a.wait_ns)) {
                    break;
                }
                tc_fence_after();
                loaded = __shfl_sync(FULL, loaded, 0);
                if (any && a.residual != nullptr && warp_wait(bar, (loaded - 1u) & 1u, abort_word, a.wait_ns)) {
                    break;
                }
                for (uint32_t c = 0; any && c < live; c += 16u) {
                    uint32_t q[16];
                    float v[16], r[16];
                    tmem_ld16(from + c, q);
#pragma unroll
                    for (uint32_t j = 0; j < 16u; ++j) {
                        r[j] = 0.0f;
                        if (a.residual != nullptr) {
                            uint16_t x;
                            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(x) : "r"(mine + (c + j) * 64u));
                            r[j] = __uint_as_float((uint32_t)x << 16);
                        }
                    }
                    tmem_ld_wait();
#pragma unroll
                    for (uint32_t j = 0; j < 16u; ++j) {
                        v[j] = __uint_as_float(q[j]);
                    }
                    finish_sums(a, o, scales, c, v, r);
#pragma unroll
                    for (uint32_t j = 0; j < 16u; ++j) {
                        asm volatile("st.shared.u16 [%0], %1;" ::"r"(mine + (c + j) * 64u), "h"(__bfloat16_as_ushort(__float2bfloat16_rn(v[j])))
                                     : "memory");
                    }
                }
                if (any) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0u) {
                        tma_store_2d(&a.out_map, mine, (int32_t)n, (int32_t)token0);
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    }
                }
            } else {
                float r[16];
                residuals_of(a, o, token0, n, live, r);
                if (warp_wait(base + S::ACC_FULL + 8 * b, turn / S::ACCS & 1u, abort_word, a.wait_ns)) {
                    break;
                }
                tc_fence_after();
                for (uint32_t c = 0; c < live; c += 16u) {
                    uint32_t q[16];
                    float v[16], next[16];
                    tmem_ld16(from + c, q);
                    residuals_of(a, o, token0 + c + 16u, n, live > c + 16u ? live - c - 16u : 0u, next);  // (asked for a round ahead)
                    tmem_ld_wait();
#pragma unroll
                    for (uint32_t j = 0; j < 16u; ++j) {
                        v[j] = __uint_as_float(q[j]);
                    }
                    finish(a, o, scales, c, token0 + c, n, live - c, v, r);
#pragma unroll
                    for (uint32_t j = 0; j < 16u; ++j) {
                        r[j] = next[j];
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0u) {
                asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(
                                 at_rank(base + S::ACC_EMPTY + 8 * b, first))
                             : "memory");
            }
        }
        // (Nothing is on its way to or from this block's shared memory when it ends: outs here; residuals that
        // nobody waited for, if it has given up.)
        if (lane == 0u) {
            asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            if (*abort_word && loaded > 0u) {
                mbar_drain(base + S::RESIDUAL + 8 * (warp - 2u), (loaded - 1u) & 1u, a.wait_ns);
            }
        }
        __syncwarp();
    }
    if (a.shares > 1u) {
        // One tile a cluster: every pair has multiplied its share of the columns for all of the tile's tokens; it
        // gets the others' sums of its part of the tokens, adds them up in the order of the shares, and
        // finishes them. The sums lie over the stages, which nobody needs by then.
        const uint32_t quad = warp % 4u, half = (warp - 2u) / 4u, row = quad * 32u + lane;
        const uint32_t n = pair / a.token_tiles * S::TILE + rank * TILE_M + row;
        const uint32_t per = a.tile_tokens / a.shares;
        const auto part_at = [&](uint32_t from, uint32_t c) { return base + ((from * (per / 4u) + c / 4u) * TILE_M + row) * 16u; };
        const uint32_t begin = half * (per / 2u), token0 = pair % a.token_tiles * a.tile_tokens;
        const uint32_t mine = token0 + share * per + begin;  // this warp's tokens
        const uint32_t live = mine < a.tokens ? min(per / 2u, a.tokens - mine) : 0u;
        Output o = {1.0f, 0.0f, false};
        const TokenScales scales(a, mine, epilogue ? live : 0u);
        float r[8];
        bool there = false;
        if (epilogue) {
            o = output_of(a, n);
            residuals_of(a, o, mine, n, live, r);
            there = !warp_wait(base + S::ACC_FULL, 0u, abort_word, a.wait_ns);
        }
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        if (there) {
            tc_fence_after();
            for (uint32_t c = half * 16u; c < a.tile_tokens; c += 32u) {
                uint32_t q[16];
                tmem_ld16(tmem + (quad * 32u << 16) + c, q);
                tmem_ld_wait();
#pragma unroll
                for (uint32_t j = 0; j < 16u; j += 4u) {
                    const uint32_t to = (c + j) / per;
                    asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(
                                     at_rank(part_at(share, c + j - to * per), 2u * to + rank)),
                                 "r"(q[j]), "r"(q[j + 1u]), "r"(q[j + 2u]), "r"(q[j + 3u])
                                 : "memory");
                }
            }
        }
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        if (there) {
            for (uint32_t c = 0; c < live; c += 8u) {
                float v[8] = {}, next[8];
                residuals_of(a, o, mine + c + 8u, n, live > c + 8u ? live - c - 8u : 0u, next);
                for (uint32_t k = 0; k < a.shares; ++k) {
#pragma unroll
                    for (uint32_t j = 0; j < 8u; j += 4u) {
                        const float4 p = *reinterpret_cast<const float4 *>(smem + (part_at(k, begin + c + j) - base));
                        v[j] += p.x, v[j + 1u] += p.y, v[j + 2u] += p.z, v[j + 3u] += p.w;
                    }
                }
                finish(a, o, scales, c, mine + c, n, live - c, v, r);
#pragma unroll
                for (uint32_t j = 0; j < 8u; ++j) {
                    r[j] = next[j];
                }
            }
        }
        __syncwarp();
    }

    if (rank == 1u && tid == 64u) {
        mbar_drain(base + S::FINAL, 0u, a.wait_ns);  // (the last commit arrives in this block, too, before it ends)
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_arrive();
    cluster_wait();  // (neither block's barriers and tensor memory go while the other may use them)
    if (*abort_word) {  // (a block's copies are counted at its pair's first block's barriers: that one has given up, too)
        stay_for_landings();
    }
    tc_fence_after();
    if (warp == 1u) {
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::COLS) : "memory");
    }
    if (tid == 0 && *abort_word) {
        atomicOr(a.status_word, 1u << lily_head::STATUS_TIMEOUT_BIT);
    }
}

template <uint32_t N, bool E4M3>
cudaError_t launch_few(const LinearArgs &a, uint32_t blocks, uint32_t shares, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks, 1, 1);
    cfg.blockDim = dim3(Few<N>::THREADS, 1, 1);
    cfg.dynamicSmemBytes = Few<N>::BYTES;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = shares;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, linear_few_kernel<N, E4M3>, a);
}

// How many clusters of 1 << i pairs run at once, asked once for a device. Not all SMs of a part of it fit into
// clusters: 74, 33 and 15 of 148 SMs. One tile more than that waits for all the others (300 x 4096 x 2048, sixteen
// tiles: four shares 25.8 us, two 14.8).
template <bool E4M3>
cudaError_t clusters_at_once(uint64_t (&most)[3]) {
    static std::atomic<uint32_t> known[64][3] = {};  // (plus one: 0 is not known)
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    for (uint32_t i = 0; e == cudaSuccess && i < 3u; ++i) {
        std::atomic<uint32_t> &mine = known[device & 63][i];
        uint32_t seen = mine.load(std::memory_order_relaxed);
        if (seen == 0u) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(2u << i, 1, 1);
            cfg.blockDim = dim3(Many::THREADS, 1, 1);
            cfg.dynamicSmemBytes = Many::BYTES;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = 2u << i;
            attr[0].val.clusterDim.y = 1;
            attr[0].val.clusterDim.z = 1;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            int found = 0;
            e = cudaOccupancyMaxActiveClusters(&found, linear_many_kernel<E4M3>, &cfg);
            seen = (uint32_t)found + 1u;
            if (e == cudaSuccess) {
                mine.store(seen, std::memory_order_relaxed);
            }
        }
        most[i] = seen - 1u;
    }
    return e;
}

template <bool E4M3>
cudaError_t launch_many(const LinearArgs &a, uint32_t clusters, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2u * a.shares * clusters, 1, 1);
    cfg.blockDim = dim3(Many::THREADS, 1, 1);
    cfg.dynamicSmemBytes = Many::BYTES;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 2u * a.shares;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, linear_many_kernel<E4M3>, a);
}

template <bool E4M3>
cudaError_t few_by_tokens(const LinearArgs &a, uint32_t n, uint32_t blocks, uint32_t shares, cudaStream_t stream) {
    return n == 16u           ? launch_few<16, E4M3>(a, blocks, shares, stream)
           : n == 32u || E4M3 ? launch_few<32, E4M3>(a, blocks, shares, stream)
                              : launch_few<64, false>(a, blocks, shares, stream);
}

bool encode_rows(CUtensorMap *map, const void *p, uint64_t ld, uint32_t rows, uint32_t columns, uint32_t dtype,
                 uint32_t box_rows) {
    const uint32_t size = dtype == LILY_BF16 ? 2u : 1u;
    const cuuint64_t dims[2] = {columns, rows};
    // (The pitch of a single row is never used, but has to be in order.)
    const cuuint64_t strides[1] = {rows > 1u ? ld * size : ((uint64_t)columns * size + 15u) & ~uint64_t(15)};
    const cuuint32_t box[2] = {BLOCK_BYTES / size, box_rows};
    const cuuint32_t estr[2] = {1, 1};
    return tensor_map_encoder()(map, size == 2u ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 2,
                                const_cast<void *>(p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// bf16 outs or residuals, in boxes of `tokens` x 32 outputs.
bool encode_outs(CUtensorMap *map, const void *p, uint64_t ld, const lily_linear_args_t &g, uint32_t tokens) {
    const cuuint64_t dims[2] = {g.outputs, g.tokens};
    const cuuint64_t strides[1] = {ld * 2u};
    const cuuint32_t box[2] = {32u, tokens};
    const cuuint32_t estr[2] = {1, 1};
    return tensor_map_encoder()(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void *>(p), dims, strides, box, estr,
                                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

cudaError_t lily_host::linear_ready() {
    static std::atomic<uint64_t> seen{0};
    return once_per_device(seen, [] {
        for (const cudaError_t e : {load_kernel(linear_few_kernel<16, false>, Few<16>::BYTES), load_kernel(linear_few_kernel<16, true>, Few<16>::BYTES),
                                    load_kernel(linear_few_kernel<32, false>, Few<32>::BYTES), load_kernel(linear_few_kernel<32, true>, Few<32>::BYTES),
                                    load_kernel(linear_few_kernel<64, false>, Few<64>::BYTES), load_kernel(linear_many_kernel<false>, Many::BYTES),
                                    load_kernel(linear_many_kernel<true>, Many::BYTES)}) {
            if (e != cudaSuccess) {
                return e;
            }
        }
        uint64_t most[3];
        const cudaError_t e = clusters_at_once<false>(most);
        return e != cudaSuccess ? e : clusters_at_once<true>(most);
    });
}

extern "C" int32_t lily_linear(lily_sampler_t *h, void *stream_, const lily_linear_args_t *args) {
    const int32_t st = check_handle(h);
    if (st != LILY_OK) {
        return st;
    }
    if (args == nullptr || args->struct_size != sizeof(lily_linear_args_t)) {
        return fail(h, LILY_ERR_ARG, "args is null or of another ABI version");
    }
    const lily_linear_args_t &g = *args;
    constexpr uint32_t MOST = 1u << 30;  // (coordinates of copies are 32 bits, signed)
    if (g.tokens == 0u || g.columns == 0u || g.outputs == 0u || g.tokens > MOST || g.columns > MOST || g.outputs > MOST) {
        return fail(h, LILY_ERR_CAPACITY, "tokens, columns and outputs must be 1..2^30");
    }
    if (g.a == nullptr || g.weight == nullptr || g.out == nullptr) {
        return fail(h, LILY_ERR_ARG, "a, weight and out must be set");
    }
    if ((g.dtype != LILY_BF16 && g.dtype != LILY_E4M3) || g.out_dtype > LILY_BF16 || g.bias_dtype > LILY_BF16 ||
        g.activation > LILY_ACT_GELU_TANH) {
        return fail(h, LILY_ERR_ARG, "a and weight are BF16 or E4M3, out and bias F32 or BF16, activation one of the five");
    }
    const bool e4m3 = g.dtype == LILY_E4M3;
    if ((g.a_scales != nullptr) != e4m3 || (g.weight_scales != nullptr) != e4m3) {
        return fail(h, LILY_ERR_ARG, "a_scales and weight_scales go with E4M3, and only with it");
    }
    if (g.a_ld < g.columns || g.weight_ld < g.columns || g.out_ld < g.outputs ||
        (g.residual != nullptr && g.residual_ld < g.outputs)) {
        return fail(h, LILY_ERR_ARG, "a row pitch is smaller than its row");
    }
    const uint32_t size = e4m3 ? 1u : 2u, out_size = g.out_dtype == LILY_F32 ? 4u : 2u;
    if (reinterpret_cast<uintptr_t>(g.a) % 16u || reinterpret_cast<uintptr_t>(g.weight) % 16u ||
        (g.tokens > 1u && g.a_ld * size % 16u) || (g.outputs > 1u && g.weight_ld * size % 16u)) {
        return fail(h, LILY_ERR_ARG, "rows of a and weight must start on 16-byte boundaries");
    }
    if ((g.tokens > 1u && g.a_ld * size >> 40) || (g.outputs > 1u && g.weight_ld * size >> 40)) {
        return fail(h, LILY_ERR_CAPACITY, "a row pitch beyond 2^40 bytes");
    }
    if (reinterpret_cast<uintptr_t>(g.out) % out_size || reinterpret_cast<uintptr_t>(g.residual) % out_size ||
        reinterpret_cast<uintptr_t>(g.bias) % (g.bias_dtype == LILY_F32 ? 4u : 2u) ||
        reinterpret_cast<uintptr_t>(g.a_scales) % 4u || reinterpret_cast<uintptr_t>(g.weight_scales) % 4u) {
        return fail(h, LILY_ERR_ARG, "a buffer is not aligned to its elements");
    }
    if (g.residual == g.out && g.residual_ld != g.out_ld) {
        return fail(h, LILY_ERR_ARG, "in place means the same pitch");
    }
    if (tensor_map_encoder() == nullptr) {
        return fail(h, LILY_ERR_CUDA, "the driver does not offer cuTensorMapEncodeTiled");
    }
    DeviceGuard guard(h->device);
    LinearArgs a;
    a.a_scales = g.a_scales, a.w_scales = g.weight_scales;
    a.bias = g.bias, a.residual = g.residual, a.out = g.out;
    a.residual_ld = g.residual_ld, a.out_ld = g.out_ld;
    a.tokens = g.tokens, a.outputs = g.outputs;
    a.blocks = (uint32_t)(((uint64_t)g.columns * size + BLOCK_BYTES - 1u) / BLOCK_BYTES);
    a.out_f32 = g.out_dtype == LILY_F32, a.bias_f32 = g.bias_dtype == LILY_F32, a.activation = g.activation;
    a.status_word = h->status_word, a.wait_ns = h->wait_ns;
    a.lost_stage = h->lost_stage;
    h->lost_stage = 0xFFFFFFFFu;  // one launch only

    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    const uint64_t sms = (uint32_t)h->sm_count;
    // By pairs from 65 tokens on; from 33 unless the weights are bf16 and their tiles more than pairs (64 x 4096 x 11000:
    // 20.7 us, by single blocks 23.0; 64 x 8192 x 2048 11.6 and 14.9; e4m3 33 x 2048 x 151936 53 and 67; the other way
    // 64 x 2048 x 20000 21.3 and 19.9, 64 x 2048 x 151936 104 and 101).
    if (g.tokens > 64u || (g.tokens > 32u && (e4m3 || (g.outputs + Many::TILE - 1ull) / Many::TILE <= sms / 2u))) {
        const auto rows16 = [&](const void *p, uint64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16u == 0u && ld * 2u % 16u == 0u; };
        // (A copy out of shared memory writes whole 16 bytes: rows of 1003 outputs had zeroes behind them.)
        const bool copies = !a.out_f32 && g.outputs % 8u == 0u && rows16(g.out, g.out_ld) &&
                            (g.residual == nullptr || rows16(g.residual, g.residual_ld));
        // The tile's tokens and the shares of its columns, by the time of the busiest pair, in units of which 1900
        // are a microsecond. A step takes the longest of its multiplies (256 tokens 0.27 us), of what all pairs
        // read (256 + t rows of 128 bytes each, 11.5 TB/s together), of a copy's way (1.35 us) by the stages there are, and of
        // asking for its copies (0.18 us). A tile's end costs by its tokens (16 ns each), joining shares by the sums that
        // are sent (two of 256 tokens 5 us). (512 x 4096 x 4096 e4m3, without the copies' way: tiles of 192 tokens for
        // 128, 15.4 us for 13.0.)
        uint64_t most[3] = {};
        CU(h, e4m3 ? clusters_at_once<true>(most) : clusters_at_once<false>(most));
        const uint64_t pairs = most[0], output_tiles = (g.outputs + Many::TILE - 1ull) / Many::TILE;
        if (pairs == 0u) {
            return fail(h, LILY_ERR_CUDA, "the device has no room for a pair of blocks");
        }
        uint64_t best = ~0ull;
        for (uint32_t t = Many::TILE; t >= 64u; t -= 32u) {
            const uint64_t tiles = (g.tokens + t - 1u) / t * output_tiles;
            for (uint32_t i = 0, shares = 1u; i < 3u; ++i, shares *= 2u) {
                if (shares > 1u && (tiles > most[i] || a.blocks < 8u * shares || t % (16u * shares) != 0u)) {
                    continue;
                }
                const uint32_t stages = Many::stages_of(t, copies && shares == 1u);
                const uint64_t steps = (tiles + pairs - 1u) / pairs * ((a.blocks + shares - 1u) / shares);
                const uint64_t step = std::max<uint64_t>({2u * t, (256u + t) * std::min(tiles * shares, pairs) * 2u / 95u, 2565u / stages, 340u});
                const uint64_t cost = steps * step + t / shares * 31u + (shares > 1u ? t * (shares - 1u) / shares * 70u + 1000u : 0u);
                if (cost < best) {
                    best = cost;
                    a.tile_tokens = t, a.shares = shares, a.stages = stages, a.copies = copies && shares == 1u;
                }
            }
        }
        a.token_tiles = (g.tokens + a.tile_tokens - 1u) / a.tile_tokens;
        const uint64_t tiles = a.token_tiles * output_tiles;
        if (tiles > 0x7FFFFFFFull) {
            return fail(h, LILY_ERR_CAPACITY, "more tiles than a launch takes");
        }
        if (!encode_rows(&a.w_map, g.weight, g.weight_ld, g.outputs, g.columns, g.dtype, TILE_M) ||
            !encode_rows(&a.a_map, g.a, g.a_ld, g.tokens, g.columns, g.dtype, a.tile_tokens / 2u) ||
            (a.copies && (!encode_outs(&a.out_map, g.out, g.out_ld, g, a.tile_tokens / 2u) ||
                          (g.residual != nullptr && !encode_outs(&a.residual_map, g.residual, g.residual_ld, g, a.tile_tokens / 2u))))) {
            return fail(h, LILY_ERR_CUDA, "cuTensorMapEncodeTiled refused a, weight, out or residual");
        }
        const uint32_t used = (uint32_t)std::min(tiles, pairs);  // (with shares, fewer tiles than pairs)
        CU(h, e4m3 ? launch_many<true>(a, used, stream) : launch_many<false>(a, used, stream));
        return LILY_OK;
    }
    const uint32_t n = g.tokens <= 16u ? 16u : g.tokens <= 32u ? 32u : 64u;
    // Shares of the columns: as many blocks as there are SMs, of four steps at least; up to 32 tokens two on an SM, of
    // eight (24 x 4096 x 4096: e4m3, four shares of eight steps 7.7 us, eight of four 8.2; bf16, of sixteen 10.6, of
    // eight 9.4).
    uint64_t tiles = (g.outputs + TILE_M - 1ull) / TILE_M;
    uint32_t shares = 8u;
    while (shares > 1u && (tiles * shares > sms * (n <= 32u ? 2u : 1u) ||
                           a.blocks < (tiles * shares > sms ? 8u : 4u) * shares)) {
        shares /= 2u;
    }
    // A tile's outputs, where blocks have tiles of their own: those of which the busiest block is done first. A step
    // takes the longest of its weights' rows (6.5 TB/s for all blocks together), of these and the tokens', which every
    // tile reads again (11 TB/s), and of a copy's way (1.35 us) by the stages there are.
    const auto stages_of = [n](uint32_t outputs) {
        return n == 16u ? Few<16>::stages_of(outputs) : n == 32u ? Few<32>::stages_of(outputs) : Few<64>::stages_of(outputs);
    };
    a.tile_outputs = TILE_M;
    if (shares == 1u) {
        uint64_t best = ~0ull;
        for (uint32_t rows = TILE_M; rows >= 48u; rows -= 8u) {
            const uint64_t count = (g.outputs + rows - 1ull) / rows, active = std::min(count, 2u * sms);
            const uint64_t step = std::max<uint64_t>({rows * 10u * active / (2u * sms), (rows + n) * 6u * active / (2u * sms), 2310u / stages_of(rows)});
            const uint64_t cost = (count + 2u * sms - 1u) / (2u * sms) * step;
            if (cost < best) {
                best = cost;
                a.tile_outputs = rows;
            }
        }
        tiles = (g.outputs + a.tile_outputs - 1ull) / a.tile_outputs;
    }
    a.stages = stages_of(a.tile_outputs);
    if (!encode_rows(&a.w_map, g.weight, g.weight_ld, g.outputs, g.columns, g.dtype, a.tile_outputs) ||
        !encode_rows(&a.a_map, g.a, g.a_ld, g.tokens, g.columns, g.dtype, n)) {
        return fail(h, LILY_ERR_CUDA, "cuTensorMapEncodeTiled refused a or weight");
    }
    const uint32_t blocks = (uint32_t)std::min<uint64_t>(tiles, sms * 2u) * shares;
    CU(h, e4m3 ? few_by_tokens<true>(a, n, blocks, shares, stream) : few_by_tokens<false>(a, n, blocks, shares, stream));
    return LILY_OK;
}
