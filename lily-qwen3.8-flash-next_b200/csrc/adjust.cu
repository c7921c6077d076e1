// Biases, penalties, bans and grammar masks written onto logits (lily_adjust_logits,
// include/lily_sampler.h).
//
// A row is cut into slices of the vocabulary, a block each. A block marks in shared memory what the
// row's lists say about its own ids (the whole lists are read by every slice: they come out of L2),
// then passes over its logits once. Blocks have nothing to say to one another, so nothing is kept
// between calls and no workspace is needed. A logit that the mask takes away is not read, and in
// place one that nothing changes is neither read nor written.
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>
#include <cstdio>
#include <cstring>

#include "../../include/lily_sampler.h"
#include "handle.cuh"

namespace {

using namespace lily_host;

constexpr uint32_t NT = 512;
constexpr uint32_t MOST_SMEM = 100u * 1024u;  // of a block: two on an SM
constexpr uint32_t NO_SLOT = 0xFFFFFFFFu;

struct RowPenalty {
    float repetition, presence, frequency;
    uint32_t slot;
};

struct AdjustArgs {
    const void *logits;
    void *out;
    uint64_t logits_ld, out_ld;
    const lily_sampling_params_t *params;  // on the device, or null
    const uint32_t *history_ids, *history_len;
    const uint32_t *bias_ids, *bias_len;
    const float *bias_vals;
    const uint32_t *ban_ids, *ban_len;
    const uint32_t *mask;
    const int32_t *mask_rows;
    uint64_t history_ld, bias_ld, ban_ld, mask_ld;
    const uint32_t *counts_table, *seen_table;
    uint32_t seen_words;
    uint32_t *out_status, *status_word;
    uint32_t row0, vocab, first_id, slice_len, masks, max_history, max_list;
    uint32_t in_place;
    uint32_t wide_counts;   // 32 bits a count: lists that can hold an id more than 65535 times
    uint32_t room_counts;   // whether the block has room for counts at all
};

// The penalties of a launch's rows travel in its arguments.
template <uint32_t MAX_ROWS>
struct AdjustLaunch {
    AdjustArgs a;
    RowPenalty rows[MAX_ROWS];
};

__device__ __forceinline__ float neg_inf() { return __uint_as_float(0xFF800000u); }

// What the block's shared memory says about an id of its slice.
struct Marks {
    const uint32_t *seen, *biased, *banned;
    const void *counts;
};

// A row as its block sees it.
struct Row {
    float repetition, presence, frequency;
    bool penalties, counted, listed_bias, listed_ban;
    const uint32_t *slot_seen, *slot_counts;  // the histogram slot's, from the slice's first id on
    const uint32_t *bias_ids;
    const float *bias_vals;
    uint32_t bias_len;
    const uint32_t *mask;   // the row's words, or null
    uint32_t id0;           // global id of the slice's first logit
};

// The 32 bits of a row of words from bit `bit` on; only words that hold one of the `n` wanted bits are read.
__device__ __forceinline__ uint32_t bits_at(const uint32_t *words, uint32_t bit, uint32_t n) {
    const uint32_t w = bit / 32u, s = bit % 32u;
    const uint32_t lo = __ldg(words + w);
    const uint32_t hi = s + n > 32u ? __ldg(words + w + 1u) : 0u;
    return __funnelshift_r(lo, hi, s);
}

__device__ __forceinline__ uint32_t count_of(const AdjustArgs &a, const Marks &m, const Row &r, uint32_t at) {
    if (r.slot_seen != nullptr) {
        return __ldg(r.slot_counts + at);
    }
    return a.wide_counts ? static_cast<const uint32_t *>(m.counts)[at] : static_cast<const uint16_t *>(m.counts)[at];
}

// Logit `x` of place `at` of the slice, biased and penalised as the marks say.
__device__ __forceinline__ float adjusted(const AdjustArgs &a, const Marks &m, const Row &r, uint32_t at, float x,
                                          bool seen, bool biased) {
    if (biased) {
        for (uint32_t j = 0; j < r.bias_len; ++j) {
            if (__ldg(r.bias_ids + j) == r.id0 + at) {
                x = __fadd_rn(x, __ldg(r.bias_vals + j));
            }
        }
    }
    if (seen) {
        const float count = r.counted ? (float)count_of(a, m, r, at) : 1.0f;
        if (count > 0.0f) {
            x = x > 0.0f ? __fdiv_rn(x, r.repetition) : __fmul_rn(x, r.repetition);
            x = __fsub_rn(x, __fadd_rn(r.presence, __fmul_rn(r.frequency, count)));
        }
    }
    return x;
}

// Which of the 32 ids of word `w` of the slice have been seen, biased, and may be drawn; n of them exist.
__device__ __forceinline__ void words_of(const Marks &m, const Row &r, uint32_t w, uint32_t n, uint32_t &seen,
                                         uint32_t &biased, uint32_t &allowed) {
    seen = !r.penalties ? 0u : r.slot_seen != nullptr ? __ldg(r.slot_seen + w) : m.seen[w];
    biased = r.listed_bias ? m.biased[w] : 0u;
    allowed = r.mask != nullptr ? bits_at(r.mask, r.id0 + w * 32u, n) : 0xFFFFFFFFu;
    if (r.listed_ban) {
        allowed &= ~m.banned[w];
    }
}

__device__ __forceinline__ float widen(float f) { return f; }
__device__ __forceinline__ float widen(__nv_bfloat16 b) { return __bfloat162float(b); }
__device__ __forceinline__ void narrow(float *to, float f) { *to = f; }
__device__ __forceinline__ void narrow(__nv_bfloat16 *to, float f) { *to = __float2bfloat16_rn(f); }

// Eight logits as they lie in memory.
template <typename T>
struct Raw;
template <>
struct Raw<float> {
    float4 a, b;
};
template <>
struct Raw<__nv_bfloat16> {
    uint4 q;
};

__device__ __forceinline__ void load8(const float *p, Raw<float> &r) {
    r.a = __ldcs(reinterpret_cast<const float4 *>(p)), r.b = __ldcs(reinterpret_cast<const float4 *>(p) + 1);
}
__device__ __forceinline__ void load8(const __nv_bfloat16 *p, Raw<__nv_bfloat16> &r) {
    r.q = __ldcs(reinterpret_cast<const uint4 *>(p));
}

__device__ __forceinline__ void unpack(const Raw<float> &r, float (&f)[8]) {
    f[0] = r.a.x, f[1] = r.a.y, f[2] = r.a.z, f[3] = r.a.w, f[4] = r.b.x, f[5] = r.b.y, f[6] = r.b.z, f[7] = r.b.w;
}
__device__ __forceinline__ void unpack(const Raw<__nv_bfloat16> &r, float (&f)[8]) {
    const uint32_t w[4] = {r.q.x, r.q.y, r.q.z, r.q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}

__device__ __forceinline__ void store8(float *p, const float (&f)[8]) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}

__device__ __forceinline__ void store8(__nv_bfloat16 *p, const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t *>(&b);
    }
    *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// What the row's lists say about the slice, into shared memory (cleared before).
__device__ __forceinline__ void mark(uint32_t *words, uint32_t at) { atomicOr(words + at / 32u, 1u << (at % 32u)); }

// TI: the logits' type, TO: out's. WIDE: rows start on 16-byte boundaries in both.
template <typename TI, typename TO, bool WIDE, uint32_t MAX_ROWS>
__global__ void __launch_bounds__(NT, 2) adjust_logits_kernel(const __grid_constant__ AdjustLaunch<MAX_ROWS> l) {
    extern __shared__ __align__(16) uint32_t smem[];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const AdjustArgs &a = l.a;
    const uint32_t t = threadIdx.x, row = a.row0 + blockIdx.y;
    const uint32_t lo = blockIdx.x * a.slice_len, n = min(a.slice_len, a.vocab - lo);

    // The row's parameters and lengths, and whether they are in order.
    Row r;
    uint32_t slot = NO_SLOT, status = LILY_ROW_OK;
    r.repetition = 1.0f, r.presence = 0.0f, r.frequency = 0.0f;
    if (a.params != nullptr) {
        const lily_sampling_params_t &p = a.params[row];
        r.repetition = p.repetition_penalty, r.presence = p.presence_penalty, r.frequency = p.frequency_penalty;
        const bool fine = isfinite(p.temperature) && p.temperature >= 0.0f && isfinite(p.top_p) && p.top_p > 0.0f &&
                          p.top_p <= 1.0f && isfinite(p.min_p) && p.min_p >= 0.0f && p.min_p <= 1.0f &&
                          isfinite(r.repetition) && r.repetition > 0.0f && isfinite(r.presence) && isfinite(r.frequency);
        status = fine ? status : LILY_ROW_PARAMS;
    }
    if (MAX_ROWS > 1u) {
        const RowPenalty &p = l.rows[blockIdx.y];
        slot = p.slot;
        if (a.params == nullptr) {
            r.repetition = p.repetition, r.presence = p.presence, r.frequency = p.frequency;
        }
    }
    r.penalties = r.presence != 0.0f || r.frequency != 0.0f || r.repetition != 1.0f;
    uint32_t history = 0, ban_len = 0;
    r.bias_len = 0;
    if (a.history_ids != nullptr && slot == NO_SLOT) {
        history = a.history_len[row];
        status = history > a.max_history || history > a.history_ld ? LILY_ROW_LIST : status;
    }
    if (a.bias_ids != nullptr) {
        r.bias_len = a.bias_len[row];
        status = r.bias_len > a.max_list || r.bias_len > a.bias_ld ? LILY_ROW_LIST : status;
    }
    if (a.ban_ids != nullptr) {
        ban_len = a.ban_len[row];
        status = ban_len > a.max_list || ban_len > a.ban_ld ? LILY_ROW_LIST : status;
    }
    int32_t mask_row = a.mask != nullptr ? (a.mask_rows != nullptr ? a.mask_rows[row] : (int32_t)row) : -1;
    status = mask_row >= 0 && (uint32_t)mask_row >= a.masks ? LILY_ROW_LIST : status;
    if (blockIdx.x == 0u && t == 0u) {
        if (a.out_status != nullptr) {
            a.out_status[row] = status;
        }
        if (status != LILY_ROW_OK) {
            atomicOr(a.status_word, 1u << status);
        }
    }
    if (status != LILY_ROW_OK) {
        return;
    }
    history = r.penalties ? history : 0u;
    r.penalties = r.penalties && (history > 0u || slot != NO_SLOT);
    r.counted = slot != NO_SLOT || r.frequency != 0.0f;
    r.listed_bias = r.bias_len > 0u;
    r.listed_ban = ban_len > 0u;
    r.id0 = a.first_id + lo;
    r.mask = mask_row >= 0 ? a.mask + (uint64_t)mask_row * a.mask_ld : nullptr;
    r.bias_ids = a.bias_ids + (uint64_t)row * a.bias_ld;
    r.bias_vals = a.bias_vals + (uint64_t)row * a.bias_ld;
    r.slot_seen = r.slot_counts = nullptr;
    if (slot != NO_SLOT) {
        r.slot_seen = a.seen_table + (uint64_t)slot * a.seen_words + lo / 32u;
        r.slot_counts = a.counts_table + (uint64_t)slot * a.vocab + lo;
    }

    // Marks: three words of bits per 32 ids, then the counts of a row with a frequency penalty.
    const uint32_t words = a.slice_len / 32u;
    uint32_t *seen = smem, *biased = smem + words, *banned = smem + 2u * words, *counts = smem + 3u * words;
    const bool own_counts = history > 0u && r.counted;
    const bool marks = history > 0u || r.listed_bias || r.listed_ban;
    if (marks) {
        const uint32_t clear = 3u * words + (own_counts ? (a.wide_counts ? a.slice_len : a.slice_len / 2u) : 0u);
        for (uint32_t i = t * 4u; i < clear; i += NT * 4u) {  // (slices are multiples of 256 ids)
            *reinterpret_cast<uint4 *>(smem + i) = make_uint4(0u, 0u, 0u, 0u);
        }
        __syncthreads();
        const uint32_t *ids = a.history_ids + (uint64_t)row * a.history_ld;
        const auto mark_history = [&](uint32_t id) {
            const uint32_t at = id - r.id0;  // (ids below the slice wrap around)
            if (at < n) {
                mark(seen, at);
                if (own_counts) {
                    if (a.wide_counts) {
                        atomicAdd(counts + at, 1u);
                    } else {
                        atomicAdd(counts + at / 2u, at % 2u ? 0x10000u : 1u);
                    }
                }
            }
        };
        const uint32_t head = min(history, (uint32_t)((16u - (reinterpret_cast<uintptr_t>(ids) & 15u)) & 15u) / 4u);
        const uint32_t quads = (history - head) / 4u;
        const uint4 *four = reinterpret_cast<const uint4 *>(ids + head);
        for (uint32_t q = t; q < quads; q += NT * 4u) {
            uint4 v[4];
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k) {
                if (q + k * NT < quads) {
                    v[k] = __ldg(four + q + k * NT);
                }
            }
#pragma unroll
            for (uint32_t k = 0; k < 4u; ++k) {
                if (q + k * NT < quads) {
                    mark_history(v[k].x), mark_history(v[k].y), mark_history(v[k].z), mark_history(v[k].w);
                }
            }
        }
        if (t < head) {
            mark_history(__ldg(ids + t));
        }
        if (head + 4u * quads + t < history) {
            mark_history(__ldg(ids + head + 4u * quads + t));
        }
        for (uint32_t j = t; j < r.bias_len; j += NT) {
            const uint32_t at = __ldg(r.bias_ids + j) - r.id0;
            if (at < n) {
                mark(biased, at);
            }
        }
        const uint32_t *ban_ids = a.ban_ids + (uint64_t)row * a.ban_ld;
        for (uint32_t j = t; j < ban_len; j += NT) {
            const uint32_t at = __ldg(ban_ids + j) - r.id0;
            if (at < n) {
                mark(banned, at);
            }
        }
        __syncthreads();
    }
    const Marks m = {seen, biased, banned, counts};

    const TI *from = static_cast<const TI *>(a.logits) + (uint64_t)row * a.logits_ld + lo;
    TO *to = static_cast<TO *>(a.out) + (uint64_t)row * a.out_ld + lo;
    if (WIDE) {
        // A thread takes eight neighbours, a quarter of a word of marks, at a time.
        constexpr uint32_t AHEAD = sizeof(TI) == 2 ? 4u : 2u;
        const uint32_t chunks = n / 8u;
        for (uint32_t c0 = t; c0 < chunks; c0 += NT * AHEAD) {
            Raw<TI> raw[AHEAD];
            uint32_t said[AHEAD];  // seen, biased, allowed, a byte each; bit 24: something is written
#pragma unroll
            for (uint32_t k = 0; k < AHEAD; ++k) {
                const uint32_t c = c0 + k * NT;
                said[k] = 0u;
                if (c < chunks) {
                    uint32_t s, b, w;
                    const uint32_t word = c / 4u, shift = c % 4u * 8u;
                    words_of(m, r, word, min(32u, n - word * 32u), s, b, w);
                    s = (s >> shift) & 0xFFu, b = (b >> shift) & 0xFFu, w = (w >> shift) & 0xFFu;
                    if (!a.in_place || w != 0xFFu || (s | b) != 0u) {
                        said[k] = s | b << 8 | w << 16 | 1u << 24;
                        if (w != 0u) {
                            load8(from + c * 8u, raw[k]);
                        }
                    }
                }
            }
#pragma unroll
            for (uint32_t k = 0; k < AHEAD; ++k) {
                const uint32_t c = c0 + k * NT;
                if (said[k] == 0u) {
                    continue;
                }
                const uint32_t s = said[k] & 0xFFu, b = said[k] >> 8 & 0xFFu, w = said[k] >> 16 & 0xFFu;
                float f[8];
                unpack(raw[k], f);
                for (uint32_t left = (s | b) & w; left != 0u; left &= left - 1u) {
                    const uint32_t i = __ffs(left) - 1u;
                    float x = 0.0f;
#pragma unroll
                    for (uint32_t j = 0; j < 8u; ++j) {
                        x = i == j ? f[j] : x;
                    }
                    x = adjusted(a, m, r, c * 8u + i, x, s >> i & 1u, b >> i & 1u);
#pragma unroll
                    for (uint32_t j = 0; j < 8u; ++j) {
                        f[j] = i == j ? x : f[j];
                    }
                }
#pragma unroll
                for (uint32_t i = 0; i < 8u; ++i) {
                    f[i] = w >> i & 1u ? f[i] : neg_inf();
                }
                store8(to + c * 8u, f);
            }
        }
    }
    // One logit a thread, a warp per word of marks: rows that start anywhere, and a wide row's last
    // few logits.
    constexpr uint32_t AHEAD = 6u;
    const uint32_t begin = WIDE ? n / 8u * 8u : 0u;
    for (uint32_t i0 = begin / 32u * 32u + t; i0 < n; i0 += NT * AHEAD) {
        float f[AHEAD];
        bool seen1[AHEAD], biased1[AHEAD], allowed1[AHEAD], any[AHEAD];
#pragma unroll
        for (uint32_t k = 0; k < AHEAD; ++k) {
            const uint32_t i = i0 + k * NT;
            any[k] = false;
            if (i < n && i >= begin) {
                uint32_t s, b, w;
                words_of(m, r, i / 32u, min(32u, n - i / 32u * 32u), s, b, w);
                seen1[k] = s >> (i % 32u) & 1u, biased1[k] = b >> (i % 32u) & 1u, allowed1[k] = w >> (i % 32u) & 1u;
                any[k] = !(a.in_place && allowed1[k] && !seen1[k] && !biased1[k]);
                if (any[k] && allowed1[k]) {
                    f[k] = widen(from[i]);
                }
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < AHEAD; ++k) {
            const uint32_t i = i0 + k * NT;
            if (any[k]) {
                if (!allowed1[k]) {
                    f[k] = neg_inf();
                } else if (seen1[k] || biased1[k]) {
                    f[k] = adjusted(a, m, r, i, f[k], seen1[k], biased1[k]);
                }
                narrow(to + i, f[k]);
            }
        }
    }
}

template <typename TI, typename TO, bool WIDE, uint32_t MAX_ROWS>
cudaError_t launch_adjust(const AdjustLaunch<MAX_ROWS> &l, uint32_t slices, uint32_t rows, size_t smem, cudaStream_t stream) {
    auto kernel = adjust_logits_kernel<TI, TO, WIDE, MAX_ROWS>;
    if (smem > 48u * 1024u) {
        static std::atomic<uint64_t> ready{0};  // (bit d: device d knows)
        int device = 0;
        cudaError_t e = cudaGetDevice(&device);
        const uint64_t bit = 1ull << (device & 63);
        if (e == cudaSuccess && !(ready.load(std::memory_order_relaxed) & bit)) {
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)MOST_SMEM);
            ready.fetch_or(e == cudaSuccess ? bit : 0u, std::memory_order_relaxed);
        }
        if (e != cudaSuccess) {
            return e;
        }
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(slices, rows, 1);
    cfg.blockDim = dim3(NT, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, l);
}

template <uint32_t MAX_ROWS>
cudaError_t adjust_by_type(const AdjustLaunch<MAX_ROWS> &l, uint32_t in, uint32_t out, bool wide, uint32_t slices,
                           uint32_t rows, size_t smem, cudaStream_t stream) {
    using B = __nv_bfloat16;
    if (in == LILY_F32) {
        return wide ? launch_adjust<float, float, true>(l, slices, rows, smem, stream)
                    : launch_adjust<float, float, false>(l, slices, rows, smem, stream);
    }
    if (out == LILY_F32) {
        return wide ? launch_adjust<B, float, true>(l, slices, rows, smem, stream)
                    : launch_adjust<B, float, false>(l, slices, rows, smem, stream);
    }
    return wide ? launch_adjust<B, B, true>(l, slices, rows, smem, stream)
                : launch_adjust<B, B, false>(l, slices, rows, smem, stream);
}

// The rows [row0, row0 + rows) of a call, their penalties and slots in the launch's arguments.
template <uint32_t MAX_ROWS>
cudaError_t adjust_rows(const AdjustArgs &a, const lily_adjust_args_t &g, uint32_t row0, uint32_t rows, bool wide,
                        uint32_t slices, size_t smem, cudaStream_t stream) {
    AdjustLaunch<MAX_ROWS> l;
    l.a = a;
    l.a.row0 = row0;
    if (MAX_ROWS > 1u) {
        for (uint32_t i = 0; i < rows && i < MAX_ROWS; ++i) {
            RowPenalty &p = l.rows[i];
            p = {1.0f, 0.0f, 0.0f, g.count_slots != nullptr ? g.count_slots[row0 + i] : NO_SLOT};
            if (g.params != nullptr && !g.params_on_device) {
                const lily_sampling_params_t &q = g.params[row0 + i];
                p.repetition = q.repetition_penalty, p.presence = q.presence_penalty, p.frequency = q.frequency_penalty;
            }
        }
    }
    return adjust_by_type(l, g.logits_dtype, g.out_dtype, wide, slices, rows, smem, stream);
}

constexpr uint32_t ROWS_FEW = 16, ROWS_MANY = 256;

}  // namespace

extern "C" int32_t lily_adjust_logits(lily_sampler_t *h, void *stream_, const lily_adjust_args_t *args) {
    const int32_t st = check_handle(h);
    if (st != LILY_OK) {
        return st;
    }
    if (args == nullptr || args->struct_size != sizeof(lily_adjust_args_t)) {
        return fail(h, LILY_ERR_ARG, "args is null or of another ABI version");
    }
    const lily_adjust_args_t &g = *args;
    if (g.rows == 0u || g.rows > h->max_rows) {
        return fail(h, LILY_ERR_CAPACITY, "rows outside 1..max_rows");
    }
    if (g.logits == nullptr || g.out == nullptr || g.logits_ld < h->vocab || g.out_ld < h->vocab ||
        g.logits_dtype > LILY_BF16 || (g.out_dtype != g.logits_dtype && g.out_dtype != LILY_F32)) {
        return fail(h, LILY_ERR_ARG, "logits must be F32 or BF16 [rows, ld >= vocab], out of that type or F32");
    }
    const uint32_t in_size = g.logits_dtype == LILY_F32 ? 4u : 2u, out_size = g.out_dtype == LILY_F32 ? 4u : 2u;
    if (reinterpret_cast<uintptr_t>(g.logits) % in_size || reinterpret_cast<uintptr_t>(g.out) % out_size) {
        return fail(h, LILY_ERR_ARG, "logits or out is not aligned to its elements");
    }
    const bool in_place = g.out == g.logits;
    if (in_place && (g.out_dtype != g.logits_dtype || (g.rows > 1u && g.out_ld != g.logits_ld))) {
        return fail(h, LILY_ERR_ARG, "in place means the same type and pitch");
    }
    if ((g.history_ids != nullptr) != (g.history_len != nullptr) || (g.bias_ids != nullptr) != (g.bias_len != nullptr) ||
        (g.bias_ids != nullptr) != (g.bias_vals != nullptr) || (g.ban_ids != nullptr) != (g.ban_len != nullptr)) {
        return fail(h, LILY_ERR_ARG, "a list needs both its ids and its lengths");
    }
    if ((uint64_t)g.first_id + h->vocab > 0xFFFFFFFFull) {
        return fail(h, LILY_ERR_ARG, "first_id + vocab overflows an id");
    }
    if (g.mask != nullptr && (g.mask_ld * 32u < (uint64_t)g.first_id + h->vocab || g.masks == 0u ||
                              (g.mask_rows == nullptr && g.masks < g.rows))) {
        return fail(h, LILY_ERR_ARG, "masks of at least first_id + vocab bits, one per row if mask_rows is NULL");
    }
    if (g.mask == nullptr && g.mask_rows != nullptr) {
        return fail(h, LILY_ERR_ARG, "mask_rows without mask");
    }
    if (g.count_slots != nullptr && (h->counts_table == nullptr || g.first_id != 0u)) {
        return fail(h, LILY_ERR_ARG, "count_slots needs LILY_FLAG_COUNTS_TABLE and first_id 0");
    }
    bool counts = g.params != nullptr && g.params_on_device, penalties = counts;
    for (uint32_t r = 0; r < g.rows; ++r) {
        if (g.params != nullptr && !g.params_on_device) {
            if (!params_ok(g.params[r])) {
                char buf[64];
                std::snprintf(buf, sizeof buf, "row %u: invalid sampling parameters", r);
                return fail(h, LILY_ERR_PARAMS, buf);
            }
            counts = counts || g.params[r].frequency_penalty != 0.0f;
            penalties = penalties || counts || g.params[r].presence_penalty != 0.0f || g.params[r].repetition_penalty != 1.0f;
        }
        if (g.count_slots != nullptr && g.count_slots[r] >= h->max_rows) {
            return fail(h, LILY_ERR_ARG, "no such histogram slot");
        }
    }
    DeviceGuard guard(h->device);
    AdjustArgs a;
    std::memset(&a, 0, sizeof a);
    a.logits = g.logits, a.out = g.out, a.logits_ld = g.logits_ld, a.out_ld = g.out_ld;
    a.params = g.params_on_device ? g.params : nullptr;
    const bool history = penalties && g.history_ids != nullptr && g.count_slots == nullptr;
    a.history_ids = g.history_ids, a.history_len = g.history_len, a.history_ld = g.history_ld;
    a.bias_ids = g.bias_ids, a.bias_vals = g.bias_vals, a.bias_len = g.bias_len, a.bias_ld = g.bias_ld;
    a.ban_ids = g.ban_ids, a.ban_len = g.ban_len, a.ban_ld = g.ban_ld;
    a.mask = g.mask, a.mask_ld = g.mask_ld, a.mask_rows = g.mask_rows, a.masks = g.masks;
    a.counts_table = h->counts_table, a.seen_table = h->seen_table, a.seen_words = h->seen_words;
    a.out_status = g.out_status, a.status_word = h->status_word;
    a.vocab = h->vocab, a.first_id = g.first_id, a.max_history = h->max_history, a.max_list = h->max_list;
    a.in_place = in_place ? 1u : 0u;
    a.wide_counts = std::min<uint64_t>(g.history_ld, h->max_history) > 65535u ? 1u : 0u;

    // Slices: enough blocks to fill the device, of shared memory that leaves room for two on an SM.
    counts = counts && history;
    const uint32_t per_id8 = 3u + (counts ? (a.wide_counts ? 32u : 16u) : 0u);  // bits of shared memory an id
    const uint32_t most = (MOST_SMEM * 8u / per_id8) & ~255u;
    const uint32_t want = std::max(1u, (2u * (uint32_t)h->sm_count + g.rows - 1u) / g.rows);
    const uint32_t least = 4096u;
    uint32_t slice = std::min(most, std::max(least, (h->vocab + want - 1u) / want));
    slice = (slice + 255u) & ~255u;
    uint32_t slices = (h->vocab + slice - 1u) / slice;
    a.slice_len = slice;
    const bool lists = history || g.bias_ids != nullptr || g.ban_ids != nullptr;
    const size_t smem = lists ? (size_t)slice * per_id8 / 8u : 0u;

    const auto rows16 = [&](const void *p, uint64_t ld, uint32_t size) {
        return reinterpret_cast<uintptr_t>(p) % 16u == 0u && (g.rows == 1u || ld * size % 16u == 0u);
    };
    const bool wide = rows16(g.logits, g.logits_ld, in_size) && rows16(g.out, g.out_ld, out_size);
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    const bool plain = (g.params == nullptr || g.params_on_device) && g.count_slots == nullptr;
    const uint32_t step = plain ? 32768u : ROWS_MANY;  // (a grid has at most 65535 rows)
    for (uint32_t r = 0; r < g.rows; r += step) {
        const uint32_t rows = std::min(step, g.rows - r);
        if (plain) {
            CU(h, adjust_rows<1>(a, g, r, rows, wide, slices, smem, stream));
        } else if (rows <= ROWS_FEW) {
            CU(h, adjust_rows<ROWS_FEW>(a, g, r, rows, wide, slices, smem, stream));
        } else {
            CU(h, adjust_rows<ROWS_MANY>(a, g, r, rows, wide, slices, smem, stream));
        }
    }
    return LILY_OK;
}
