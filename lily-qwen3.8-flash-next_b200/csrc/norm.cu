// The residual's addition and the root-mean-square norm (lily_add_rms_norm, include/lily_layers.h).
//
// A token is one thread block's, held in registers from its loads to its stores, so that x and
// the residual are read once and h and out written once: 7 bytes a value with a bf16 residual and
// 8-bit codes, and nothing else of size. One reduction serves both statistics: with u = h * weight,
// y = u / rms, so the largest |y| is the largest |u| over rms, and the 8-bit codes need no
// second round through the block; they are those of y as the other types get it, rounded to binary32.
//
// What bounds it: memory from a few hundred tokens on (16384 x 4096 bf16 to codes 72 to 77 us with
// its residual, 6.5 to 6.1 TB/s; 777 x 5001 f32 8.2 us, out of L2 in part); below, the launch and one way through a block:
// 1.5 us on the device, 3 through a Python call.
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
    uint32_t tokens, hidden, weight_f32;
    float inv_hidden, eps, offset;
};

// How a row's values are dealt out to its threads, eight to a vector.
enum Deal {
    ALIGNED,   // rows start on 16-byte boundaries and are a multiple of eight values long: neighbours
    SHIFTED,   // rows start anywhere, but all tensors' rows alike: neighbours from the boundary before the row's start
    SCATTERED  // anything else: a block's width apart
};

// A thread's vector j of a row: the place of its first value (below 0 before a shifted row's start).
template <Deal D, uint32_t WIDTH>
struct Vector {
    int32_t first;
    uint32_t step;
    __device__ __forceinline__ Vector(uint32_t j, uint32_t shift) {
        const uint32_t width = WIDTH ? WIDTH : blockDim.x, t = WIDTH ? threadIdx.x % (WIDTH ? WIDTH : 1u) : threadIdx.x;
        first = D == SCATTERED ? (int32_t)(j * width * V + t) : (int32_t)((j * width + t) * V) - (int32_t)shift;
        step = D == SCATTERED ? width : 1u;
    }
    // Whether some of its values are the row's; whether all of them are, next to one another.
    __device__ __forceinline__ bool some(uint32_t n) const { return first < (int32_t)n; }
    __device__ __forceinline__ bool all(uint32_t n) const {
        return D == ALIGNED || (D == SHIFTED && first >= 0 && first + (int32_t)V <= (int32_t)n);
    }
    __device__ __forceinline__ bool has(uint32_t k, uint32_t n) const {
        return (uint32_t)(first + (int32_t)(k * step)) < n;
    }
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

template <typename T, typename Vec>
__device__ __forceinline__ void load(const T *row, const Vec &v, uint32_t n, Raw<T> &r) {
    if (v.some(n)) {
        if (v.all(n)) {
            r = *reinterpret_cast<const Raw<T> *>(row + v.first);
        } else {
#pragma unroll
            for (uint32_t k = 0; k < V; ++k) {
                if (v.has(k, n)) {
                    set(r, k, row[v.first + (int32_t)(k * v.step)]);
                }
            }
        }
    }
}

// The weights of a vector, 0 where it has none. `weight` starts on a 16-byte boundary unless the deal is
// SCATTERED; a shifted vector's lie in two of its vectors.
template <typename W, Deal D, typename Vec>
__device__ __forceinline__ void weights(const W *weight, const Vec &v, uint32_t n, uint32_t shift, float (&f)[V]) {
    Raw<W> r = {};
    if (D == SHIFTED && shift != 0u && v.all(n) && v.first + (int32_t)shift + (int32_t)V <= (int32_t)n) {
        float lo[V], hi[V];
        const W *at = weight + v.first + (int32_t)shift;
        unpack(*reinterpret_cast<const Raw<W> *>(at - V), lo);
        unpack(*reinterpret_cast<const Raw<W> *>(at), hi);
        // f[k] = both[V - shift + k]: by eight, four, two and one, as the shift's bits say.
        float both[2 * V];
#pragma unroll
        for (uint32_t k = 0; k < V; ++k) {
            both[k] = lo[k];
            both[V + k] = hi[k];
        }
        const uint32_t by = V - shift;
#pragma unroll
        for (uint32_t bit = V / 2u; bit > 0u; bit /= 2u) {
#pragma unroll
            for (uint32_t k = 0; k + bit < 2u * V; ++k) {
                both[k] = by & bit ? both[k + bit] : both[k];
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < V; ++k) {
            f[k] = both[k];
        }
        return;
    }
    if (D == SHIFTED && shift != 0u && v.all(n)) {  // (the last whole vector: its second half would end past the weights)
#pragma unroll
        for (uint32_t k = 0; k < V; ++k) {
            set(r, k, weight[v.first + (int32_t)k]);
        }
    } else {
        load<W>(weight, v, n, r);
    }
    unpack(r, f);
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

template <typename T, typename Vec>
__device__ __forceinline__ void store(T *row, const Vec &v, uint32_t n, const float (&f)[V]) {
    if (v.some(n)) {
        if (v.all(n)) {
            put(row + v.first, f);
        } else {
#pragma unroll
            for (uint32_t k = 0; k < V; ++k) {
                if (v.has(k, n)) {
                    put_one(row + v.first + (int32_t)(k * v.step), f[k]);
                }
            }
        }
    }
}

// T: x's type, O: out's; VECS vectors a thread. WARPS 0: a block per token; else a warp per token,
// WARPS of them in a block. Values past a row's ends are 0 in registers.
template <typename T, typename O, uint32_t VECS, Deal D, uint32_t WARPS>
__global__ void __launch_bounds__(WARPS ? 32u * WARPS : VECS == 1u ? 1024u : 512u) add_rms_norm_kernel(const __grid_constant__ NormArgs a) {
    __shared__ float part_sum[32];
    __shared__ uint32_t part_max[32];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    constexpr bool CODES = sizeof(O) == 1;
    using Vec = Vector<D, WARPS ? 32u : 0u>;
    const uint32_t t = threadIdx.x, n = a.hidden;
    const uint64_t token = WARPS ? blockIdx.x * WARPS + t / 32u : blockIdx.x;
    if (WARPS && token >= a.tokens) {
        return;
    }
    const T *x_row = static_cast<const T *>(a.x) + token * a.x_ld;
    const uint32_t shift = D == SHIFTED ? (uint32_t)(reinterpret_cast<uintptr_t>(x_row) / sizeof(T)) % V : 0u;
    // All of it is asked for before any of it is used, as far as the registers hold it.
    constexpr bool EARLY = VECS * sizeof(T) <= 8;
    Raw<T> x[VECS] = {}, residual[EARLY ? VECS : 1] = {};
#pragma unroll
    for (uint32_t j = 0; j < VECS; ++j) {
        load<T>(x_row, Vec(j, shift), n, x[j]);
    }
    const T *residual_row = static_cast<const T *>(a.residual) + token * a.residual_ld;
    if (EARLY && a.residual != nullptr) {
#pragma unroll
        for (uint32_t j = 0; j < VECS; ++j) {
            load<T>(residual_row, Vec(j, shift), n, residual[j]);
        }
    }
    float w[EARLY ? VECS : 1][V];
    const auto weights_of = [&](uint32_t j, float (&f)[V]) {
        if (a.weight_f32) {
            weights<float, D>(static_cast<const float *>(a.weight), Vec(j, shift), n, shift, f);
        } else {
            weights<__nv_bfloat16, D>(static_cast<const __nv_bfloat16 *>(a.weight), Vec(j, shift), n, shift, f);
        }
    };
    if (EARLY) {
#pragma unroll
        for (uint32_t j = 0; j < VECS; ++j) {
            weights_of(j, w[j]);
        }
    }
    T *residual_out = static_cast<T *>(a.residual_out) + token * a.residual_out_ld;
    // h becomes u = h * weight on the way; the largest |u| by its bits, in which a NaN is above all.
    float u[VECS][V], sum = 0.0f;
    uint32_t largest = 0u;
#pragma unroll
    for (uint32_t j = 0; j < VECS; ++j) {
        unpack(x[j], u[j]);
        if (a.residual != nullptr) {
            float f[V];
            if (!EARLY) {
                load<T>(residual_row, Vec(j, shift), n, residual[0] = {});
            }
            unpack(residual[EARLY ? j : 0], f);
#pragma unroll
            for (uint32_t k = 0; k < V; ++k) {
                u[j][k] += f[k];
            }
        }
        if (a.residual_out != nullptr) {
            store<T>(residual_out, Vec(j, shift), n, u[j]);
        }
        if (!EARLY) {
            weights_of(j, w[0]);
        }
#pragma unroll
        for (uint32_t k = 0; k < V; ++k) {
            sum = fmaf(u[j][k], u[j][k], sum);
            u[j][k] *= a.offset + w[EARLY ? j : 0][k];
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
    if (WARPS == 0u) {
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
        if (CODES) {
            largest = __reduce_max_sync(0xFFFFFFFFu, lane < warps ? part_max[lane] : 0u);
        }
    }
    const float factor = 1.0f / sqrtf(fmaf(sum, a.inv_hidden, a.eps));
    float to_codes = 1.0f;
    if (CODES) {
        float m = __uint_as_float(largest) * factor;  // (rounding keeps the order: this is the largest |y|, rounded)
        m = m < 0x1p-64f ? 0x1p-64f : m;              // (a NaN stays)
        if (WARPS ? lane == 0u : t == 0u) {
            a.out_scales[token] = m / E4M3_MAX;
        }
        to_codes = E4M3_MAX / m;
    }
    O *out = static_cast<O *>(a.out) + token * a.out_ld;
#pragma unroll
    for (uint32_t j = 0; j < VECS; ++j) {
#pragma unroll
        for (uint32_t k = 0; k < V; ++k) {
            // (Not by factor * to_codes: that product rounds apart, 1e-5 of the codes came out beside those of y, and can
            // pass the format's range where neither step does.)
            u[j][k] = CODES ? u[j][k] * factor * to_codes : u[j][k] * factor;
        }
        store<O>(out, Vec(j, shift), n, u[j]);
    }
}

constexpr uint32_t NORM_WARPS = 8;  // of a block whose warps have a token each

template <typename T, typename O, uint32_t VECS, Deal D, uint32_t WARPS>
cudaError_t launch_norm(const NormArgs &a, cudaStream_t stream) {
    const uint32_t per = V * VECS, values = a.hidden + (D == SHIFTED ? V - 1u : 0u);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(WARPS ? (a.tokens + WARPS - 1u) / (WARPS ? WARPS : 1u) : a.tokens, 1, 1);
    cfg.blockDim = dim3(WARPS ? 32u * WARPS : (((values + per - 1u) / per) + 31u) & ~31u, 1, 1);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, add_rms_norm_kernel<T, O, VECS, D, WARPS>, a);
}

template <typename T, typename O>
cudaError_t norm_by_size(const NormArgs &a, Deal deal, bool many, cudaStream_t stream) {
    constexpr uint32_t WARPS = NORM_WARPS;
    if (deal == SCATTERED) {
        return a.hidden <= 8192u ? launch_norm<T, O, 1, SCATTERED, 0>(a, stream) : launch_norm<T, O, 8, SCATTERED, 0>(a, stream);
    }
    // Many short rows: a warp each, with nothing to wait for (16384 x 512 bf16 to codes 17.5 -> 10.4 us, floor 9.0).
    if (many && deal == ALIGNED && a.hidden <= 1024u) {
        return a.hidden <= 256u   ? launch_norm<T, O, 1, ALIGNED, WARPS>(a, stream)
               : a.hidden <= 512u ? launch_norm<T, O, 2, ALIGNED, WARPS>(a, stream)
                                  : launch_norm<T, O, 4, ALIGNED, WARPS>(a, stream);
    }
    // Few tokens (two blocks an SM or less): as many threads as there are vectors, the shortest way
    // through a block. Many: blocks of 256 threads or so, whose loads in flight come from several vectors a thread:
    // 16384 x 4096 bf16 to codes 77.3 us with one vector a thread, 72.0 with two and 72.5 with four (floor
    // 71.8); 8000 x 8192 f32 to codes 69.4, 66.2 and 51.7 (50.1). A row that misses the boundaries costs a
    // tenth more than one that does not (777 x 5001 and 5008 f32: 9.8 and 9.0 us, scattered 15.7).
    const uint32_t vectors = (a.hidden + (deal == SHIFTED ? 2u * V - 2u : V - 1u)) / V, threads = many ? 256u : 1024u;
    const uint32_t vecs = vectors > 2048u ? 8u : vectors > std::min(1024u, 2u * threads) ? 4u : vectors > threads ? 2u : 1u;
    if (deal == ALIGNED) {
        return vecs == 8u   ? launch_norm<T, O, 8, ALIGNED, 0>(a, stream)
               : vecs == 4u ? launch_norm<T, O, 4, ALIGNED, 0>(a, stream)
               : vecs == 2u ? launch_norm<T, O, 2, ALIGNED, 0>(a, stream)
                            : launch_norm<T, O, 1, ALIGNED, 0>(a, stream);
    }
    return vecs == 8u   ? launch_norm<T, O, 8, SHIFTED, 0>(a, stream)
           : vecs == 4u ? launch_norm<T, O, 4, SHIFTED, 0>(a, stream)
           : vecs == 2u ? launch_norm<T, O, 2, SHIFTED, 0>(a, stream)
                        : launch_norm<T, O, 1, SHIFTED, 0>(a, stream);
}

template <typename T>
cudaError_t norm_by_out(const NormArgs &a, uint32_t out_dtype, Deal deal, bool many, cudaStream_t stream) {
    return out_dtype == LILY_F32    ? norm_by_size<T, float>(a, deal, many, stream)
           : out_dtype == LILY_BF16 ? norm_by_size<T, __nv_bfloat16>(a, deal, many, stream)
                                    : norm_by_size<T, __nv_fp8_e4m3>(a, deal, many, stream);
}

// The variants that norm_by_size chooses from.
template <typename T, typename O>
cudaError_t load_norms() {
    constexpr uint32_t W = NORM_WARPS;
    for (const cudaError_t e : {load_kernel(add_rms_norm_kernel<T, O, 1, SCATTERED, 0>), load_kernel(add_rms_norm_kernel<T, O, 8, SCATTERED, 0>),
                                load_kernel(add_rms_norm_kernel<T, O, 1, ALIGNED, W>), load_kernel(add_rms_norm_kernel<T, O, 2, ALIGNED, W>),
                                load_kernel(add_rms_norm_kernel<T, O, 4, ALIGNED, W>), load_kernel(add_rms_norm_kernel<T, O, 1, ALIGNED, 0>),
                                load_kernel(add_rms_norm_kernel<T, O, 2, ALIGNED, 0>), load_kernel(add_rms_norm_kernel<T, O, 4, ALIGNED, 0>),
                                load_kernel(add_rms_norm_kernel<T, O, 8, ALIGNED, 0>), load_kernel(add_rms_norm_kernel<T, O, 1, SHIFTED, 0>),
                                load_kernel(add_rms_norm_kernel<T, O, 2, SHIFTED, 0>), load_kernel(add_rms_norm_kernel<T, O, 4, SHIFTED, 0>),
                                load_kernel(add_rms_norm_kernel<T, O, 8, SHIFTED, 0>)}) {
        if (e != cudaSuccess) {
            return e;
        }
    }
    return cudaSuccess;
}

template <typename T>
cudaError_t load_norms_of() {
    for (const cudaError_t e : {load_norms<T, float>(), load_norms<T, __nv_bfloat16>(), load_norms<T, __nv_fp8_e4m3>()}) {
        if (e != cudaSuccess) {
            return e;
        }
    }
    return cudaSuccess;
}

uint32_t element(uint32_t dtype) { return dtype == LILY_F32 ? 4u : dtype == LILY_BF16 ? 2u : 1u; }

// Whether rows of `ld` elements all start on multiples of `bytes`.
bool rows_at(const void *p, uint64_t ld, uint32_t dtype, uint32_t rows, uint32_t bytes) {
    return p == nullptr ||
           (reinterpret_cast<uintptr_t>(p) % bytes == 0u && (rows == 1u || ld * element(dtype) % bytes == 0u));
}

}  // namespace

cudaError_t lily_host::norm_ready() {
    static std::atomic<uint64_t> seen{0};
    return once_per_device(seen, [] {
        const cudaError_t e = load_norms_of<float>();
        return e != cudaSuccess ? e : load_norms_of<__nv_bfloat16>();
    });
}

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
    a.tokens = g.tokens, a.weight_f32 = g.weight_dtype == LILY_F32;
    // The deal: rows 16 bytes at a time where they allow it, or where all of them miss a boundary of
    // eight values alike.
    Deal deal = SCATTERED;
    if (reinterpret_cast<uintptr_t>(g.weight) % 16u == 0u) {
        const auto miss = [&](const void *p, uint32_t dtype) { return (uint32_t)(reinterpret_cast<uintptr_t>(p) / element(dtype) % V); };
        const auto alike = [&](const void *p, uint64_t ld, uint32_t dtype) {
            return p == nullptr || (miss(p, dtype) == miss(g.x, g.dtype) && (g.tokens == 1u || ld % V == g.x_ld % V));
        };
        if (alike(g.residual, g.residual_ld, g.dtype) && alike(g.residual_out, g.residual_out_ld, g.dtype) &&
            alike(g.out, g.out_ld, g.out_dtype)) {
            deal = g.hidden % V == 0u && miss(g.x, g.dtype) == 0u && (g.tokens == 1u || g.x_ld % V == 0u) ? ALIGNED : SHIFTED;
        }
    }
    if (deal == SHIFTED && g.hidden > LILY_NORM_MAX_HIDDEN - V) {
        deal = SCATTERED;  // (a shifted row takes one vector more than the largest block's threads have)
    }
    const bool many = g.tokens > 2u * (uint32_t)h->sm_count;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    CU(h, g.dtype == LILY_F32 ? norm_by_out<float>(a, g.out_dtype, deal, many, s)
                              : norm_by_out<__nv_bfloat16>(a, g.out_dtype, deal, many, s));
    return LILY_OK;
}
