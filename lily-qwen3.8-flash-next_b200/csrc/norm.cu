// The residual's addition and the root-mean-square norm (lily_add_rms_norm, include/lily_layers.h).
//
// A token is one thread block's, held in registers from its loads to its stores, so that x and
// the residual are read once and h and out written once: 7 bytes a value with a bf16 residual and
// 8-bit codes, and nothing else of size. One reduction serves both statistics: with u = h * weight,
// y = u / rms, so the largest |y| is the largest |u| over rms, and the 8-bit codes need no
// second round through the block.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>

#include "../../include/lily_layers.h"
#include "handle.cuh"

namespace {

using namespace lily_host;

constexpr uint32_t V = 8;  // values of a vector: 16 bytes of bf16, 32 of f32
constexpr float E4M3_MAX = 448.0f;

struct NormArgs {
    const void *x, *residual, *weight;
    void *residual_out, *out;
    float *out_scales;
    uint64_t x_ld, residual_ld, residual_out_ld, out_ld;
    uint32_t hidden;
    float inv_hidden, eps, offset;
};

template <typename T>
struct Raw;  // V values as they lie in memory
template <>
struct Raw<float> {
    float4 q[2];
};
template <>
struct Raw<__nv_bfloat16> {
    uint4 q;
};

__device__ __forceinline__ void set(Raw<float> &r, uint32_t k, float f) {
    float4 &q = r.q[k / 4u];
    (k % 4u == 0u ? q.x : k % 4u == 1u ? q.y : k % 4u == 2u ? q.z : q.w) = f;
}

__device__ __forceinline__ void set(Raw<__nv_bfloat16> &r, uint32_t k, __nv_bfloat16 b) {
    uint32_t &w = k / 2u == 0u ? r.q.x : k / 2u == 1u ? r.q.y : k / 2u == 2u ? r.q.z : r.q.w;
    w |= (uint32_t)__bfloat16_as_ushort(b) << (k % 2u * 16u);  // (from zero)
}

__device__ __forceinline__ void unpack(const Raw<float> &r, float (&f)[V]) {
    f[0] = r.q[0].x, f[1] = r.q[0].y, f[2] = r.q[0].z, f[3] = r.q[0].w;
    f[4] = r.q[1].x, f[5] = r.q[1].y, f[6] = r.q[1].z, f[7] = r.q[1].w;
}

__device__ __forceinline__ void unpack(const Raw<__nv_bfloat16> &r, float (&f)[V]) {
    const uint32_t w[4] = {r.q.x, r.q.y, r.q.z, r.q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}

// The V values of a thread's vector j of a row of n: neighbours where the rows allow it (WIDE: they
// start on 16-byte boundaries and n is a multiple of V), a block's width apart where they do not.
template <bool WIDE>
__device__ __forceinline__ uint32_t first_of(uint32_t j) {
    return WIDE ? (j * blockDim.x + threadIdx.x) * V : j * blockDim.x * V + threadIdx.x;
}

template <typename T, bool WIDE>
__device__ __forceinline__ void load(const T *row, uint32_t j, uint32_t n, Raw<T> &r) {
    const uint32_t i = first_of<WIDE>(j);
    if (WIDE) {
        if (i < n) {
            r = *reinterpret_cast<const Raw<T> *>(row + i);
        }
    } else {
#pragma unroll
        for (uint32_t k = 0; k < V; ++k) {
            if (i + k * blockDim.x < n) {
                set(r, k, row[i + k * blockDim.x]);
            }
        }
    }
}

__device__ __forceinline__ uint32_t two_bf16(float lo, float hi) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&b);
}

__device__ __forceinline__ void put(float *to, const float (&f)[V]) {
    reinterpret_cast<float4 *>(to)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4 *>(to)[1] = make_float4(f[4], f[5], f[6], f[7]);
}

__device__ __forceinline__ void put(__nv_bfloat16 *to, const float (&f)[V]) {
    *reinterpret_cast<uint4 *>(to) = make_uint4(two_bf16(f[0], f[1]), two_bf16(f[2], f[3]), two_bf16(f[4], f[5]),
                                                two_bf16(f[6], f[7]));
}

// (A value beyond the format's largest by a rounding of the scale becomes the largest.)
__device__ __forceinline__ uint32_t two_e4m3(float lo, float hi) {
    return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ void put(__nv_fp8_e4m3 *to, const float (&f)[V]) {
    *reinterpret_cast<uint2 *>(to) = make_uint2(two_e4m3(f[0], f[1]) | two_e4m3(f[2], f[3]) << 16,
                                                two_e4m3(f[4], f[5]) | two_e4m3(f[6], f[7]) << 16);
}

__device__ __forceinline__ void put_one(float *to, float f) { *to = f; }
__device__ __forceinline__ void put_one(__nv_bfloat16 *to, float f) { *to = __float2bfloat16_rn(f); }
__device__ __forceinline__ void put_one(__nv_fp8_e4m3 *to, float f) {
    to->__x = __nv_cvt_float_to_fp8(f, __NV_SATFINITE, __NV_E4M3);
}

template <typename T, bool WIDE>
__device__ __forceinline__ void store(T *row, uint32_t j, uint32_t n, const float (&f)[V]) {
    const uint32_t i = first_of<WIDE>(j);
    if (WIDE) {
        if (i < n) {
            put(row + i, f);
        }
    } else {
#pragma unroll
        for (uint32_t k = 0; k < V; ++k) {
            if (i + k * blockDim.x < n) {
                put_one(row + i + k * blockDim.x, f[k]);
            }
        }
    }
}

// T: x's type, W: the weight's, O: out's; VECS vectors a thread. Values past a row's end are 0
// in registers.
template <typename T, typename W, typename O, uint32_t VECS, bool WIDE>
__global__ void __launch_bounds__(1024) add_rms_norm_kernel(const __grid_constant__ NormArgs a) {
    __shared__ float part_sum[32];
    __shared__ uint32_t part_max[32];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    constexpr bool CODES = sizeof(O) == 1;
    const uint32_t t = threadIdx.x, n = a.hidden;
    const uint64_t token = blockIdx.x;
    // All of it is asked for before any of it is used, as far as 64 registers hold it.
    constexpr bool EARLY_RESIDUAL = VECS * sizeof(T) <= 8, EARLY_WEIGHT = VECS * (2 * sizeof(T) + sizeof(W)) <= 12;
    Raw<T> x[VECS] = {}, residual[EARLY_RESIDUAL ? VECS : 1] = {};
    Raw<W> weight[EARLY_WEIGHT ? VECS : 1] = {};
    const T *x_row = static_cast<const T *>(a.x) + token * a.x_ld;
#pragma unroll
    for (uint32_t j = 0; j < VECS; ++j) {
        load<T, WIDE>(x_row, j, n, x[j]);
    }
    const T *residual_row = static_cast<const T *>(a.residual) + token * a.residual_ld;
    if (EARLY_RESIDUAL && a.residual != nullptr) {
#pragma unroll
        for (uint32_t j = 0; j < VECS; ++j) {
            load<T, WIDE>(residual_row, j, n, residual[j]);
        }
    }
    if (EARLY_WEIGHT) {
#pragma unroll
        for (uint32_t j = 0; j < VECS; ++j) {
            load<W, WIDE>(static_cast<const W *>(a.weight), j, n, weight[j]);
        }
    }
    T *residual_out = static_cast<T *>(a.residual_out) + token * a.residual_out_ld;
    // h becomes u = h * weight on the way; the largest |u| by its bits, in which a NaN is above all.
    float u[VECS][V], sum = 0.0f;
    uint32_t largest = 0u;
#pragma unroll
    for (uint32_t j = 0; j < VECS; ++j) {
        float f[V];
        unpack(x[j], u[j]);
        if (a.residual != nullptr) {
            if (!EARLY_RESIDUAL) {
                load<T, WIDE>(residual_row, j, n, residual[0] = {});
            }
            unpack(residual[EARLY_RESIDUAL ? j : 0], f);
#pragma unroll
            for (uint32_t k = 0; k < V; ++k) {
                u[j][k] += f[k];
            }
        }
        if (a.residual_out != nullptr) {
            store<T, WIDE>(residual_out, j, n, u[j]);
        }
        if (!EARLY_WEIGHT) {
            load<W, WIDE>(static_cast<const W *>(a.weight), j, n, weight[0] = {});
        }
        unpack(weight[EARLY_WEIGHT ? j : 0], f);
#pragma unroll
        for (uint32_t k = 0; k < V; ++k) {
            sum = fmaf(u[j][k], u[j][k], sum);
            u[j][k] *= a.offset + f[k];
            if (CODES) {
                largest = max(largest, __float_as_uint(u[j][k]) & 0x7FFFFFFFu);
            }
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    }
    if (CODES) {
        largest = __reduce_max_sync(0xFFFFFFFFu, largest);
    }
    const uint32_t warps = blockDim.x / 32u, lane = t % 32u;
    if (lane == 0u) {
        part_sum[t / 32u] = sum;
        part_max[t / 32u] = largest;
    }
    __syncthreads();
    sum = lane < warps ? part_sum[lane] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    }
    float factor = 1.0f / sqrtf(fmaf(sum, a.inv_hidden, a.eps));
    if (CODES) {
        largest = __reduce_max_sync(0xFFFFFFFFu, lane < warps ? part_max[lane] : 0u);
        float m = __uint_as_float(largest) * factor;
        m = m < 0x1p-64f ? 0x1p-64f : m;  // (a NaN stays)
        if (t == 0u) {
            a.out_scales[token] = m / E4M3_MAX;
        }
        factor *= E4M3_MAX / m;
    }
    O *out = static_cast<O *>(a.out) + token * a.out_ld;
#pragma unroll
    for (uint32_t j = 0; j < VECS; ++j) {
#pragma unroll
        for (uint32_t k = 0; k < V; ++k) {
            u[j][k] *= factor;
        }
        store<O, WIDE>(out, j, n, u[j]);
    }
}

template <typename T, typename W, typename O, uint32_t VECS, bool WIDE>
cudaError_t launch_norm(const NormArgs &a, uint32_t tokens, cudaStream_t stream) {
    const uint32_t per = V * VECS;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(tokens, 1, 1);
    cfg.blockDim = dim3((((a.hidden + per - 1u) / per) + 31u) & ~31u, 1, 1);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, add_rms_norm_kernel<T, W, O, VECS, WIDE>, a);
}

#ifndef NORM_FEW
#define NORM_FEW 296
#endif
#ifndef NORM_MANY
#define NORM_MANY 2u
#endif
template <typename T, typename W, typename O>
cudaError_t norm_by_size(const NormArgs &a, uint32_t tokens, bool wide, cudaStream_t stream) {
    const uint32_t least = a.hidden > 16384u ? 4u : a.hidden > 8192u ? 2u : 1u;
    const uint32_t vecs = std::max(least, tokens > NORM_FEW ? NORM_MANY : 1u);
    if (vecs == 4u) {
        return wide ? launch_norm<T, W, O, 4, true>(a, tokens, stream) : launch_norm<T, W, O, 4, false>(a, tokens, stream);
    }
    if (vecs == 2u) {
        return wide ? launch_norm<T, W, O, 2, true>(a, tokens, stream) : launch_norm<T, W, O, 2, false>(a, tokens, stream);
    }
    return wide ? launch_norm<T, W, O, 1, true>(a, tokens, stream) : launch_norm<T, W, O, 1, false>(a, tokens, stream);
}

template <typename T, typename W>
cudaError_t norm_by_out(const NormArgs &a, uint32_t out_dtype, uint32_t tokens, bool wide, cudaStream_t stream) {
    return out_dtype == LILY_F32    ? norm_by_size<T, W, float>(a, tokens, wide, stream)
           : out_dtype == LILY_BF16 ? norm_by_size<T, W, __nv_bfloat16>(a, tokens, wide, stream)
                                    : norm_by_size<T, W, __nv_fp8_e4m3>(a, tokens, wide, stream);
}

template <typename T>
cudaError_t norm_by_weight(const NormArgs &a, uint32_t weight_dtype, uint32_t out_dtype, uint32_t tokens, bool wide,
                           cudaStream_t stream) {
    return weight_dtype == LILY_F32 ? norm_by_out<T, float>(a, out_dtype, tokens, wide, stream)
                                    : norm_by_out<T, __nv_bfloat16>(a, out_dtype, tokens, wide, stream);
}

uint32_t element(uint32_t dtype) { return dtype == LILY_F32 ? 4u : dtype == LILY_BF16 ? 2u : 1u; }

// Whether rows of `ld` elements all start on multiples of `bytes`.
bool rows_at(const void *p, uint64_t ld, uint32_t dtype, uint32_t rows, uint32_t bytes) {
    return p == nullptr ||
           (reinterpret_cast<uintptr_t>(p) % bytes == 0u && (rows == 1u || ld * element(dtype) % bytes == 0u));
}

}  // namespace

extern "C" int32_t lily_add_rms_norm(lily_sampler_t *h, void *stream, const lily_norm_args_t *args) {
    const int32_t st = check_handle(h);
    if (st != LILY_OK) {
        return st;
    }
    if (args == nullptr || args->struct_size != sizeof(lily_norm_args_t)) {
        return fail(h, LILY_ERR_ARG, "args is null or of another ABI version");
    }
    const lily_norm_args_t &g = *args;
    if (g.tokens == 0u || g.tokens > 0x7FFFFFFFu || g.hidden == 0u || g.hidden > LILY_NORM_MAX_HIDDEN) {
        return fail(h, LILY_ERR_CAPACITY, "tokens outside 1..2^31 - 1 or hidden outside 1..32768");
    }
    if (g.x == nullptr || g.weight == nullptr || g.out == nullptr) {
        return fail(h, LILY_ERR_ARG, "x, weight and out must be set");
    }
    if (g.dtype > LILY_BF16 || g.weight_dtype > LILY_BF16 || g.out_dtype > LILY_E4M3) {
        return fail(h, LILY_ERR_ARG, "x and weight are F32 or BF16, out F32, BF16 or E4M3");
    }
    if ((g.out_scales != nullptr) != (g.out_dtype == LILY_E4M3)) {
        return fail(h, LILY_ERR_ARG, "out_scales goes with an E4M3 out, and only with it");
    }
    if (g.x_ld < g.hidden || g.out_ld < g.hidden || (g.residual != nullptr && g.residual_ld < g.hidden) ||
        (g.residual_out != nullptr && g.residual_out_ld < g.hidden)) {
        return fail(h, LILY_ERR_ARG, "a row pitch is smaller than hidden");
    }
    if (!rows_at(g.x, g.x_ld, g.dtype, g.tokens, element(g.dtype)) ||
        !rows_at(g.residual, g.residual_ld, g.dtype, g.tokens, element(g.dtype)) ||
        !rows_at(g.residual_out, g.residual_out_ld, g.dtype, g.tokens, element(g.dtype)) ||
        !rows_at(g.out, g.out_ld, g.out_dtype, g.tokens, element(g.out_dtype)) ||
        reinterpret_cast<uintptr_t>(g.weight) % element(g.weight_dtype) != 0u ||
        reinterpret_cast<uintptr_t>(g.out_scales) % 4u != 0u) {
        return fail(h, LILY_ERR_ARG, "a buffer is not aligned to its elements");
    }
    if (!(std::isfinite(g.eps) && g.eps >= 0.0f && std::isfinite(g.weight_offset))) {
        return fail(h, LILY_ERR_ARG, "eps must be finite and not negative, weight_offset finite");
    }
    // In place: a block has read its token before it writes it, but only its own token.
    const auto clash = [&](const void *p, uint64_t ld, uint32_t dtype, const void *from, uint64_t from_ld) {
        return p != nullptr && p == from && (ld != from_ld || dtype != g.dtype);
    };
    if (clash(g.out, g.out_ld, g.out_dtype, g.x, g.x_ld) || clash(g.out, g.out_ld, g.out_dtype, g.residual, g.residual_ld) ||
        clash(g.residual_out, g.residual_out_ld, g.dtype, g.x, g.x_ld) ||
        clash(g.residual_out, g.residual_out_ld, g.dtype, g.residual, g.residual_ld) || g.out == g.residual_out) {
        return fail(h, LILY_ERR_ARG, "in place means the same pitch and type, and out is not residual_out");
    }
    DeviceGuard guard(h->device);
    NormArgs a;
    a.x = g.x, a.residual = g.residual, a.weight = g.weight;
    a.residual_out = g.residual_out, a.out = g.out, a.out_scales = g.out_scales;
    a.x_ld = g.x_ld, a.residual_ld = g.residual_ld, a.residual_out_ld = g.residual_out_ld, a.out_ld = g.out_ld;
    a.hidden = g.hidden;
    a.inv_hidden = 1.0f / (float)g.hidden;
    a.eps = g.eps, a.offset = g.weight_offset;
    const bool wide = g.hidden % V == 0u && rows_at(g.x, g.x_ld, g.dtype, g.tokens, 16u) &&
                      rows_at(g.residual, g.residual_ld, g.dtype, g.tokens, 16u) &&
                      rows_at(g.residual_out, g.residual_out_ld, g.dtype, g.tokens, 16u) &&
                      rows_at(g.out, g.out_ld, g.out_dtype, g.tokens, g.out_dtype == LILY_E4M3 ? 8u : 16u) &&
                      reinterpret_cast<uintptr_t>(g.weight) % 16u == 0u;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    CU(h, g.dtype == LILY_F32 ? norm_by_weight<float>(a, g.weight_dtype, g.out_dtype, g.tokens, wide, s)
                              : norm_by_weight<__nv_bfloat16>(a, g.weight_dtype, g.out_dtype, g.tokens, wide, s));
    return LILY_OK;
}
