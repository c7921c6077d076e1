// Biases, penalties, bans and grammar masks written onto logits (lily_adjust_logits,
// include/lily_sampler.h).
//
// Masks and bans alone are one pass over the logits: mask_logits_kernel. A logit that goes is not
// read, and in place one that stays is neither read nor written.
//
// Penalties and biases change a few thousand ids of a row, which the row's lists name: adjust_logits_kernel. A row
// is cut into slices of the vocabulary (where there are few rows; a large batch's rows are a block each),
// whose blocks' two parts work side by side: the first passes over the slice's logits as above, the second
// marks the ids of the slice that the history has, a bit each, numbers them (a prefix sum over the bits), and
// reads the history again to count them by their numbers: a few thousand counts instead of one for every
// id. When both are done, the numbered ids, which lie evenly on the threads, are penalised. Blocks have nothing
// to say to one another, so nothing is kept between calls and no workspace is needed.
//
// What bounds it: masks alone are a launch (1 x 151936 2.2 us on the device). 256 x 151936 bf16 with histories of
// 32768 ids take 58 us, 73 with masks, bans and biases, where the bytes are 26: the second part takes them (three reads
// of the ids, an atomic in shared memory for each in two of them, scattered logits at the end), and a row is one
// block's, so 256 of them fill 148 SMs unevenly. Slower there: counts of 16 bits for every id over four slices a row
// (116 us for 75 at the time), the rows' lists pulled by halves of a block (100), tasks in a pipeline (82 to 100),
// numbers handed out by atomics that return (105), parts whose threads go by the history's length (86 for 72: registers).
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>
#include <cstdio>
#include <cstring>

#include "../../include/lily_sampler.h"
#include "handle.cuh"

namespace {

using namespace lily_host;

constexpr uint32_t NO_SLOT = 0xFFFFFFFFu, NONE = 0xFFFFFFFFu, FULL = 0xFFFFFFFFu;
constexpr uint32_t MAX_LIST = 512;  // the most that a handle's max_list can be

struct RowPenalty {
    float repetition, presence, frequency;
    uint32_t slot;
};

struct AdjustArgs {
    const void *logits;
    void *out;
    uint64_t logits_ld, out_ld;
    const lily_sampling_params_t *params;  // on the device, or null
    const uint32_t *history_ids, *history_len;  // (ids null: no row of the call has penalties)
    const uint32_t *bias_ids, *bias_len;
    const float *bias_vals;
    const uint32_t *ban_ids, *ban_len;
    const uint32_t *mask;
    const int32_t *mask_rows;
    uint64_t history_ld, bias_ld, ban_ld, mask_ld;
    const uint32_t *counts_table, *seen_table;
    uint32_t seen_words;
    uint32_t *out_status, *status_word;
    uint32_t row0, rows, tasks;  // a launch's rows; rows x slices
    uint32_t vocab, first_id, slice_len, masks, max_history, max_list;
    uint32_t in_place;
    // A block's shared memory, in words from its start: bits of the ids that stay, of those in the history, how
    // many of those there are before each word of bits.
    uint32_t seen_at, before_at, direct;  // (the latter two words if not `direct`: see the kernel)
};

// The penalties of a launch's rows travel in its arguments.
template <uint32_t MAX_ROWS>
struct AdjustLaunch {
    AdjustArgs a;
    RowPenalty rows[MAX_ROWS];
};

__device__ __forceinline__ float neg_inf() { return __uint_as_float(0xFF800000u); }

// `n` bits (at most 32) of a row of words from bit `bit` on, which may lie up to 7 before its first; only
// words that hold one of them are read. What is beyond them is not defined.
__device__ __forceinline__ uint32_t bits_at(const uint32_t *words, int32_t bit, uint32_t n) {
    if (bit < 0) {
        return __ldg(words) << -bit;
    }
    const uint32_t w = (uint32_t)bit / 32u, s = (uint32_t)bit % 32u;
    const uint32_t lo = __ldg(words + w);
    const uint32_t hi = s + n > 32u ? __ldg(words + w + 1u) : 0u;
    return __funnelshift_r(lo, hi, s);
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
    uint4 q[2];
};
template <>
struct Raw<__nv_bfloat16> {
    uint4 q[1];
};

template <typename T>
__device__ __forceinline__ void load8(const T *p, Raw<T> &r) {
#pragma unroll
    for (uint32_t i = 0; i < sizeof(T) / 2u; ++i) {
        r.q[i] = __ldcs(reinterpret_cast<const uint4 *>(p) + i);
    }
}

__device__ __forceinline__ uint32_t masked(uint32_t two, uint32_t keep) {  // two bf16, by the two lowest bits of `keep`
    two = keep & 1u ? two : (two & 0xFFFF0000u) | 0xFF80u;
    return keep & 2u ? two : (two & 0xFFFFu) | 0xFF800000u;
}

// Eight logits written, -inf where `keep` has no bit.
__device__ __forceinline__ void store8(float *p, const Raw<float> &r, uint32_t keep) {
#pragma unroll
    for (uint32_t i = 0; i < 2u; ++i) {
        uint4 q = r.q[i];
        const uint32_t k = keep >> (4u * i);
        q.x = k & 1u ? q.x : 0xFF800000u, q.y = k & 2u ? q.y : 0xFF800000u;
        q.z = k & 4u ? q.z : 0xFF800000u, q.w = k & 8u ? q.w : 0xFF800000u;
        reinterpret_cast<uint4 *>(p)[i] = q;
    }
}
__device__ __forceinline__ void store8(__nv_bfloat16 *p, const Raw<__nv_bfloat16> &r, uint32_t keep) {
    uint4 q = r.q[0];
    if (keep != 0xFFu) {
        q = make_uint4(masked(q.x, keep), masked(q.y, keep >> 2), masked(q.z, keep >> 4), masked(q.w, keep >> 6));
    }
    *reinterpret_cast<uint4 *>(p) = q;
}
__device__ __forceinline__ void store8(float *p, const Raw<__nv_bfloat16> &r, uint32_t keep) {
    const uint32_t w[4] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w};
    Raw<float> f;
#pragma unroll
    for (uint32_t i = 0; i < 2u; ++i) {
        f.q[i] = make_uint4(w[2 * i] << 16, w[2 * i] & 0xFFFF0000u, w[2 * i + 1] << 16, w[2 * i + 1] & 0xFFFF0000u);
    }
    store8(p, f, keep);
}

// A row's history as a slice's block reads it: all of it. base: the id of place 0; the slice's are the `n`
// places from `shift` on.
struct HistoryList {
    const uint32_t *ids;
    uint32_t length, base, shift, n;

    // f(eight places, NONE for those that are not the slice's) over the list, by the warps of a block that
    // come here, whenever they do: they take the list's parts in turn (`next`, in shared memory, from 0), the
    // next one's ids asked for before one's are looked at.
    template <typename F>
    __device__ __forceinline__ void each(uint32_t *next, F f) const {
        constexpr uint32_t AHEAD = 4u;  // vectors of a lane in a part
        const uint32_t lane = threadIdx.x % 32u;
        const uint32_t head = min(length, (uint32_t)((16u - (reinterpret_cast<uintptr_t>(ids) & 15u)) & 15u) / 4u);
        const uint32_t quads = (length - head) / 4u, parts = (quads + 32u * AHEAD - 1u) / (32u * AHEAD);
        const uint4 *four = reinterpret_cast<const uint4 *>(ids + head);
        const auto place = [&](uint32_t id) { return id - base - shift < n ? id - base : NONE; };  // (an id below the slice wraps around)
        uint4 v[AHEAD];
        const auto take = [&]() {
            uint32_t part = 0;
            if (lane == 0u) {
                part = atomicAdd(next, 1u);
            }
            part = __shfl_sync(FULL, part, 0);
#pragma unroll
            for (uint32_t k = 0; k < AHEAD; ++k) {
                const uint32_t q = (part * AHEAD + k) * 32u + lane;
                v[k] = q < quads ? __ldg(four + q) : make_uint4(NONE, NONE, NONE, NONE);
            }
            return part;
        };
        uint32_t part = take();
        while (part < parts) {
            uint32_t p[AHEAD][4];
#pragma unroll
            for (uint32_t k = 0; k < AHEAD; ++k) {
                p[k][0] = place(v[k].x), p[k][1] = place(v[k].y), p[k][2] = place(v[k].z), p[k][3] = place(v[k].w);
            }
            part = take();
#pragma unroll
            for (uint32_t k = 0; k < AHEAD; k += 2u) {
                const uint32_t eight[8] = {p[k][0], p[k][1], p[k][2], p[k][3], p[k + 1u][0], p[k + 1u][1], p[k + 1u][2], p[k + 1u][3]};
                f(eight);
            }
        }
        if (part == parts) {  // one warp: up to three ids in front, up to three behind
            const uint32_t behind = head + 4u * quads + lane - 4u;
            const uint32_t id = lane < head ? __ldg(ids + lane) : lane >= 4u && behind < length ? __ldg(ids + behind) : NONE;
            const uint32_t eight[8] = {place(id), NONE, NONE, NONE, NONE, NONE, NONE, NONE};
            f(eight);
        }
    }
};

// Barriers of parts of a block (`threads`: those that arrive and those that wait).
constexpr uint32_t BAR_ALL = 0, BAR_STREAM = 1, BAR_LISTS = 2;
__device__ __forceinline__ void bar_sync(uint32_t bar, uint32_t threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(threads) : "memory");
}
// A task: a row's slice. WIDE: rows of logits and out start on boundaries of eight logits, or miss one
// by as much; a slice's places are then counted from the boundary before its first logit (`shift` places
// earlier), so that eight logits of a boundary are eight marks of one.
template <typename TI, typename TO, bool WIDE>
struct Task {
    const TI *from;
    TO *to;
    const uint32_t *mask;  // the row's words, or null
    float repetition, presence, frequency;
    uint32_t row, slot, history, bias_len, ban_len;
    uint32_t lo, n, id0, shift;  // the slice's first logit, its length, its first id
    uint32_t words;              // of bits, of a slice
    bool fine, penalties;

    template <uint32_t MAX_ROWS>
    __device__ __forceinline__ Task(const AdjustLaunch<MAX_ROWS> &l, uint32_t task) {
        const AdjustArgs &a = l.a;
        const uint32_t at = task % a.rows, slice = task / a.rows;
        row = a.row0 + at;
        lo = slice * a.slice_len, n = min(a.slice_len, a.vocab - lo);
        words = a.slice_len / 32u + 8u;  // (slices are multiples of 256 ids)
        uint32_t status = LILY_ROW_OK;
        slot = NO_SLOT, repetition = 1.0f, presence = 0.0f, frequency = 0.0f;
        if (a.params != nullptr) {
            const lily_sampling_params_t &p = a.params[row];
            repetition = p.repetition_penalty, presence = p.presence_penalty, frequency = p.frequency_penalty;
            const bool valid = isfinite(p.temperature) && p.temperature >= 0.0f && isfinite(p.top_p) && p.top_p > 0.0f &&
                               p.top_p <= 1.0f && isfinite(p.min_p) && p.min_p >= 0.0f && p.min_p <= 1.0f &&
                               isfinite(repetition) && repetition > 0.0f && isfinite(presence) && isfinite(frequency);
            status = valid ? status : LILY_ROW_PARAMS;
        }
        if (MAX_ROWS > 1u) {
            const RowPenalty &p = l.rows[at];
            slot = p.slot;
            if (a.params == nullptr) {
                repetition = p.repetition, presence = p.presence, frequency = p.frequency;
            }
        }
        penalties = presence != 0.0f || frequency != 0.0f || repetition != 1.0f;
        history = bias_len = ban_len = 0u;
        if (a.history_len != nullptr && slot == NO_SLOT) {
            history = a.history_len[row];
            status = history > a.max_history || history > a.history_ld ? LILY_ROW_LIST : status;
        }
        if (a.bias_ids != nullptr) {
            bias_len = a.bias_len[row];
            status = bias_len > a.max_list || bias_len > a.bias_ld ? LILY_ROW_LIST : status;
        }
        if (a.ban_ids != nullptr) {
            ban_len = a.ban_len[row];
            status = ban_len > a.max_list || ban_len > a.ban_ld ? LILY_ROW_LIST : status;
        }
        const int32_t mask_row = a.mask != nullptr ? (a.mask_rows != nullptr ? a.mask_rows[row] : (int32_t)row) : -1;
        status = mask_row >= 0 && (uint32_t)mask_row >= a.masks ? LILY_ROW_LIST : status;
        mask = mask_row >= 0 ? a.mask + (uint64_t)mask_row * a.mask_ld : nullptr;
        fine = status == LILY_ROW_OK;
        if (slice == 0u && threadIdx.x == 0u) {
            if (a.out_status != nullptr) {
                a.out_status[row] = status;
            }
            if (!fine) {
                atomicOr(a.status_word, 1u << status);
            }
        }
        history = penalties && fine && a.history_ids != nullptr ? history : 0u;
        bias_len = fine ? bias_len : 0u;
        id0 = a.first_id + lo;
        from = static_cast<const TI *>(a.logits) + (uint64_t)row * a.logits_ld + lo;
        to = static_cast<TO *>(a.out) + (uint64_t)row * a.out_ld + lo;
        shift = WIDE ? (uint32_t)(reinterpret_cast<uintptr_t>(from) / sizeof(TI)) % 8u : 0u;
    }

    __device__ __forceinline__ bool from_slot() const { return fine && penalties && slot != NO_SLOT; }
    __device__ __forceinline__ bool masks() const { return mask != nullptr || ban_len > 0u; }
    __device__ __forceinline__ bool keeps() const { return masks() || bias_len > 0u; }
    // Vectors of eight places; the first and the last may have fewer.
    __device__ __forceinline__ uint32_t chunks() const { return (n + shift + 7u) / 8u; }
    // Of the eight places from 8 c on, those that stay.
    __device__ __forceinline__ uint32_t stay8(const uint32_t *kept, uint32_t c) const {
        return keeps() ? (uint32_t)reinterpret_cast<const uint8_t *>(kept)[c] : 0xFFu;
    }

    // The slice's logits, masked and written, by `width` threads of which this is number t; what stays goes
    // into `kept`, a bit each (if anything goes, or biases have ids to take out).
    __device__ __forceinline__ void stream(const AdjustArgs &a, uint32_t *kept, uint32_t t, uint32_t width) const {
        if (keeps()) {
            if (ban_len > 0u) {
                for (uint32_t i = t; i < words; i += width) {
                    kept[i] = 0u;
                }
                bar_sync(BAR_STREAM, width);
                for (uint32_t j = t; j < ban_len; j += width) {
                    const uint32_t at = __ldg(a.ban_ids + (uint64_t)row * a.ban_ld + j) - id0;
                    if (at < n) {
                        atomicOr(kept + (at + shift) / 32u, 1u << ((at + shift) % 32u));
                    }
                }
                bar_sync(BAR_STREAM, width);
            }
            for (uint32_t i = t; i * 32u < n + shift; i += width) {
                const int32_t first = (int32_t)(i * 32u) - (int32_t)shift;
                const uint32_t stay =
                    mask != nullptr ? bits_at(mask, (int32_t)id0 + first, min(32u, (uint32_t)((int32_t)n - first))) : FULL;
                kept[i] = ban_len > 0u ? stay & ~kept[i] : stay;
            }
            bar_sync(BAR_STREAM, width);
        }
        if (a.in_place && !masks()) {
            return;
        }
        if (!WIDE) {
            for (uint32_t c = t; c < chunks(); c += width) {
                one_by_one(a, kept, c);
            }
            return;
        }
        const uint32_t begin = shift != 0u ? 1u : 0u, end = (n + shift) / 8u;  // the whole vectors
        const TI *from8 = from - shift;
        TO *to8 = to - shift;
        constexpr uint32_t AHEAD = sizeof(TI) == 2 ? 8u : 4u;
        for (uint32_t c = begin + t; c < end; c += width * AHEAD) {
            Raw<TI> raw[AHEAD];
            uint32_t keeps[AHEAD / 4u];  // a byte each
#pragma unroll
            for (uint32_t k = 0; k < AHEAD; ++k) {
                const uint32_t keep = c + k * width < end ? stay8(kept, c + k * width) : 0u;
                keeps[k / 4u] = k % 4u ? keeps[k / 4u] | keep << k % 4u * 8u : keep;
                if (keep != 0u && !(a.in_place && keep == 0xFFu)) {
                    load8(from8 + (c + k * width) * 8u, raw[k]);
                }
            }
#pragma unroll
            for (uint32_t k = 0; k < AHEAD; ++k) {
                const uint32_t keep = keeps[k / 4u] >> k % 4u * 8u & 0xFFu;
                if (c + k * width < end && !(a.in_place && keep == 0xFFu)) {
                    store8(to8 + (c + k * width) * 8u, raw[k], keep);
                }
            }
        }
        if (t == 0u && begin != 0u) {
            one_by_one(a, kept, 0u);
        }
        if (t == width - 1u && end < chunks() && (end != 0u || begin == 0u)) {
            one_by_one(a, kept, end);
        }
    }

private:
    // A vector that is not whole, or whose logits and outs do not lie alike.
    __device__ __forceinline__ void one_by_one(const AdjustArgs &a, const uint32_t *kept, uint32_t c) const {
        const int32_t first = (int32_t)(c * 8u) - (int32_t)shift;
        const uint32_t keep = stay8(kept, c);
        for (int32_t i = 0; i < 8; ++i) {
            if (first + i >= 0 && first + i < (int32_t)n) {
                if (!(keep >> i & 1u)) {
                    narrow(to + first + i, neg_inf());
                } else if (!a.in_place) {
                    narrow(to + first + i, widen(from[first + i]));
                }
            }
        }
    }
};

constexpr uint32_t MASK_NT = 512;

// Masks and bans alone. Grid: rows x slices.
template <typename TI, typename TO, bool WIDE>
__global__ void __launch_bounds__(MASK_NT, 2) mask_logits_kernel(const __grid_constant__ AdjustLaunch<1> l) {
    extern __shared__ __align__(16) uint32_t smem[];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const Task<TI, TO, WIDE> task(l, blockIdx.x);
    if (task.fine) {
        task.stream(l.a, smem, threadIdx.x, MASK_NT);
    }
}

constexpr uint32_t NT = 512;
constexpr uint32_t LISTING = 320, STREAMING = NT - LISTING;  // threads of a block's two parts
constexpr uint32_t WINDOW = 5120;  // numbered ids that a block counts at a time: what two blocks an SM leave of its shared memory

// Grid: rows x slices, the rows' first slices first.
template <typename TI, typename TO, bool WIDE, uint32_t MAX_ROWS>
__global__ void __launch_bounds__(NT, 2) adjust_logits_kernel(const __grid_constant__ AdjustLaunch<MAX_ROWS> l) {
    extern __shared__ __align__(16) uint32_t smem[];
    __shared__ uint32_t window[2u * WINDOW], sums[NT / 32u], next_part, bias_id[MAX_LIST];
    __shared__ float bias_val[MAX_LIST];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const AdjustArgs &a = l.a;
    const Task<TI, TO, WIDE> task(l, blockIdx.x);
    if (!task.fine) {
        return;
    }
    uint32_t *kept = smem, *seen = smem + a.seen_at, *before = smem + a.before_at;
    // A slice no longer than two windows needs no numbers: its places are counted as they are; so are those of
    // one of four windows, in 16 bits, if no list can have an id more often than they hold.
    const bool direct = a.direct != 0u, halves = a.direct == 2u;
    uint32_t *count_of = window, *place_of = window + WINDOW;
    const uint32_t t = threadIdx.x, lane = t % 32u, shift = task.shift;
    const uint32_t units = (task.n + shift + 31u) / 32u;  // words of bits
    const bool from_slot = task.from_slot(), history = task.history > 0u;

    // The second part finds out what the lists say while the first one passes over the logits; where a
    // short slice has a long history, both see to that together afterwards. (256 x 151936 bf16, the second part of
    // 128, 192, 256, 320 and 384 threads: 32768 ids a row 105, 81, 65, 58 and 61 us; of 256, 320 and 384: 2048 ids 36,
    // 39 and 48.) Without a history, both pass over the logits (16 biases and bans: 45 -> 36 us).
    const bool together = task.history > 2u * task.n;
    const uint32_t streaming = history ? STREAMING : NT;
    if (t < streaming) {
        task.stream(a, kept, t, streaming);
    }
    if (t >= STREAMING) {
        for (uint32_t i = t - STREAMING; history && i < (halves ? units * 16u : direct ? task.n + shift : units); i += LISTING) {
            (direct ? count_of : seen)[i] = 0u;
        }
        for (uint32_t j = t - STREAMING; j < task.bias_len; j += LISTING) {
            bias_id[j] = __ldg(a.bias_ids + (uint64_t)task.row * a.bias_ld + j);
            bias_val[j] = __ldg(a.bias_vals + (uint64_t)task.row * a.bias_ld + j);
        }
        if (t == STREAMING) {
            next_part = 0u;
        }
    }
    if (together) {
        __syncthreads();
    }
    const uint32_t width = together ? NT : LISTING, bar = together ? BAR_ALL : BAR_LISTS, me = together ? t : t - STREAMING;
    const HistoryList ids{a.history_ids + (uint64_t)task.row * a.history_ld, task.history, task.id0 - shift, shift, task.n};
    const auto mark_and_number = [&]() {
        ids.each(&next_part, [&](const uint32_t (&place)[8]) {
            // (Looked at first, all eight together: an or on a word that most of a warp means takes turns.)
            uint32_t word[8];
#pragma unroll
            for (uint32_t k = 0; k < 8u; ++k) {
                word[k] = place[k] != NONE ? reinterpret_cast<volatile uint32_t *>(seen)[place[k] / 32u] : 0xFFFFFFFFu;
            }
#pragma unroll
            for (uint32_t k = 0; k < 8u; ++k) {
                if (!(word[k] >> place[k] % 32u & 1u)) {
                    atomicOr(seen + place[k] / 32u, 1u << place[k] % 32u);
                }
            }
        });
        bar_sync(bar, width);
        // ---- numbered: what is before each word. A thread adds up neighbours.
        const uint32_t each = (units + width - 1u) / width | 1u, first = me * each;
        uint32_t mine = 0;
        for (uint32_t i = 0; i < each; ++i) {
            mine += first + i < units ? (uint32_t)__popc(seen[first + i]) : 0u;
        }
        uint32_t upto = mine;
#pragma unroll
        for (uint32_t o = 1; o < 32u; o *= 2u) {
            const uint32_t below = __shfl_up_sync(FULL, upto, o);
            upto += lane >= o ? below : 0u;
        }
        if (lane == 31u) {
            sums[me / 32u] = upto;
        }
        if (me == 0u) {
            next_part = 0u;
        }
        bar_sync(bar, width);
        uint32_t warps = lane < width / 32u ? sums[lane] : 0u;
#pragma unroll
        for (uint32_t o = 1; o < 32u; o *= 2u) {
            const uint32_t below = __shfl_up_sync(FULL, warps, o);
            warps += lane >= o ? below : 0u;
        }
        uint32_t at = upto - mine + (me >= 32u ? __shfl_sync(FULL, warps, (me / 32u + 31u) % 32u) : 0u);
        for (uint32_t i = 0; i < each && first + i < units; ++i) {
            before[first + i] = at;
            at += (uint32_t)__popc(seen[first + i]);
        }
        bar_sync(bar, width);
    };
    if (history && (together || t >= STREAMING)) {
        bar_sync(bar, width);
        // ---- the history's ids, a bit each (or their counts at once)
        if (direct) {
            ids.each(&next_part, [&](const uint32_t (&place)[8]) {
#pragma unroll
                for (uint32_t k = 0; k < 8u; ++k) {
                    if (place[k] == NONE) {
                    } else if (halves) {
                        atomicAdd(count_of + place[k] / 2u, place[k] % 2u ? 0x10000u : 1u);
                    } else {
                        atomicAdd(count_of + place[k], 1u);
                    }
                }
            });
        } else {
            mark_and_number();
        }
    }
    // Window by window: the places of the numbers from `base` on, and how often they come. (32768 ids by Zipf's law have 8000
    // to 12000 different ones, two or three windows: 256 rows 75 and 85 us, with a frequency penalty, for which every
    // window reads the history, 99 and 123.)
    const auto fill = [&](uint32_t base, uint32_t me, uint32_t width, uint32_t bar) {
        for (uint32_t i = me; i < WINDOW; i += width) {
            count_of[i] = 0u;
        }
        // (A warp's lanes look far apart: where ids are frequent, all of their neighbours are seen.)
        const uint32_t apart = (units + 31u) / 32u | 1u;
        for (uint32_t w = me / 32u; w < apart; w += width / 32u) {
            const uint32_t u = lane * apart + w;
            if (u < units) {
                uint32_t at = before[u] - base;  // (wraps around where the window begins later)
                for (uint32_t m = seen[u]; m != 0u; m &= m - 1u, ++at) {
                    if (at < WINDOW) {
                        place_of[at] = u * 32u + (uint32_t)__ffs(m) - 1u;
                    }
                }
            }
        }
        bar_sync(bar, width);
        if (task.frequency != 0.0f) {
            ids.each(&next_part, [&](const uint32_t (&place)[8]) {
                uint32_t at[8];
#pragma unroll
                for (uint32_t k = 0; k < 8u; ++k) {
                    const uint32_t u = place[k] / 32u;
                    at[k] = place[k] != NONE ? before[u] + (uint32_t)__popc(seen[u] & ((1u << place[k] % 32u) - 1u)) - base : NONE;
                }
#pragma unroll
                for (uint32_t k = 0; k < 8u; ++k) {
                    if (at[k] < WINDOW) {
                        atomicAdd(count_of + at[k], 1u);
                    }
                }
            });
        }
    };
    if (history && !direct && (together || t >= STREAMING)) {
        fill(0u, me, width, bar);
    }
    __syncthreads();  // (the logits are written, too)
    const uint32_t total = !history ? 0u : direct ? task.n + shift : before[units - 1u] + (uint32_t)__popc(seen[units - 1u]);

    const auto counted = [&](uint32_t at) -> uint32_t {
        return halves ? (uint32_t)reinterpret_cast<const uint16_t *>(count_of)[at] : count_of[at];
    };

    // ---- what the lists change
    const uint32_t *slot_seen = a.seen_table + (from_slot ? (uint64_t)task.slot * a.seen_words : 0u);
    const uint32_t *slot_counts = a.counts_table + (from_slot ? (uint64_t)task.slot * a.vocab : 0u) + task.lo;
    const auto penalised = [&](float x, uint32_t count) {
        x = x > 0.0f ? __fdiv_rn(x, task.repetition) : __fmul_rn(x, task.repetition);
        return __fsub_rn(x, __fadd_rn(task.presence, __fmul_rn(task.frequency, (float)count)));
    };
    // A biased id is its first entry's, which adds up all of them in the list's order; its penalties follow
    // where its count is known, and it no longer counts as one that stays.
    for (uint32_t j = t; j < task.bias_len; j += NT) {
        const uint32_t id = bias_id[j], in = id - task.id0, place = in + shift;
        if (in >= task.n || !(kept[place / 32u] >> place % 32u & 1u)) {
            continue;
        }
        bool first = true;
#pragma unroll 8
        for (uint32_t e = 0; e < j; ++e) {
            first = first && bias_id[e] != id;
        }
        if (first) {
            float x = widen(task.to[in]);
#pragma unroll 8
            for (uint32_t e = j; e < task.bias_len; ++e) {
                x = bias_id[e] == id ? __fadd_rn(x, bias_val[e]) : x;
            }
            if (history && (direct ? counted(place) != 0u : (seen[place / 32u] >> place % 32u & 1u) != 0u)) {
                uint32_t count = 0;
                if (direct) {
                    count = counted(place);
                } else if (task.frequency != 0.0f) {
                    const uint32_t at = before[place / 32u] + (uint32_t)__popc(seen[place / 32u] & ((1u << place % 32u) - 1u));
                    if (at < WINDOW) {
                        count = count_of[at];
                    } else {  // (a later window's: counted by itself, 0.8 ms for 32768 ids)
                        for (uint32_t i = 0; i < task.history; ++i) {
                            count += __ldg(ids.ids + i) == id ? 1u : 0u;
                        }
                    }
                }
                x = penalised(x, count);
            } else if (from_slot) {
                const uint32_t count = __ldg(slot_counts + in);
                x = count > 0u ? penalised(x, count) : x;
            }
            narrow(task.to + in, x);
        }
    }
    if (task.bias_len > 0u) {
        __syncthreads();
        for (uint32_t j = t; j < task.bias_len; j += NT) {
            const uint32_t place = bias_id[j] - task.id0 + shift;
            if (bias_id[j] - task.id0 < task.n) {
                atomicAnd(kept + place / 32u, ~(1u << place % 32u));
            }
        }
        __syncthreads();
    }
    // Values are read from `to`: the pass has just written them, they are in L2.
    constexpr uint32_t AHEAD = 8u;
    const uint32_t room = direct ? 4u * WINDOW : WINDOW;
    for (uint32_t base = 0; base < total; base += room) {
        if (base != 0u) {
            __syncthreads();
            if (t == 0u) {
                next_part = 0u;
            }
            fill(base, t, NT, BAR_ALL);
            __syncthreads();
        }
        const uint32_t held = min(room, total - base);
        for (uint32_t e = t; e < held; e += NT * AHEAD) {
            uint32_t place[AHEAD];
            float x[AHEAD];
#pragma unroll
            for (uint32_t k = 0; k < AHEAD; ++k) {
                place[k] = e + k * NT >= held ? NONE : !direct ? place_of[e + k * NT] : counted(e + k * NT) != 0u ? e + k * NT : NONE;
                if (place[k] != NONE && task.keeps() && !(kept[place[k] / 32u] >> place[k] % 32u & 1u)) {
                    place[k] = NONE;
                }
                if (place[k] != NONE) {
                    x[k] = widen(task.to[place[k] - shift]);
                }
            }
#pragma unroll
            for (uint32_t k = 0; k < AHEAD; ++k) {
                if (place[k] != NONE) {
                    narrow(task.to + place[k] - shift, penalised(x[k], counted(e + k * NT)));
                }
            }
        }
    }
    // A histogram slot's ids: its bits and counts are as they are.
    for (uint32_t u = t; from_slot && u < units; u += NT) {
        const int32_t first = (int32_t)(u * 32u) - (int32_t)shift;
        uint32_t m = bits_at(slot_seen, (int32_t)task.lo + first, min(32u, (uint32_t)((int32_t)task.n - first)));
        m &= first < 0 ? FULL << -first : FULL;  // (of the slice alone)
        m &= first + 32 > (int32_t)task.n ? FULL >> (first + 32 - (int32_t)task.n) : FULL;
        for (m &= task.keeps() ? kept[u] : FULL; m != 0u; m &= m - 1u) {
            const int32_t in = first + __ffs(m) - 1;
            const uint32_t count = __ldg(slot_counts + in);
            if (count > 0u) {
                narrow(task.to + in, penalised(widen(task.to[in]), count));
            }
        }
    }
}

constexpr uint32_t LEAST_SLICE = 2048;

// How a call is cut: slices of a row, shared memory of their blocks.
struct Cut {
    uint32_t slices;
    size_t smem;
};

// Shared memory of an adjusting block beside its window and bias entries: two on an SM.
constexpr uint32_t MOST_SMEM = 66u * 1024u;

template <typename Kernel, typename Launch>
cudaError_t launch(Kernel kernel, const Launch &l, uint32_t blocks, uint32_t threads, size_t smem, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks, 1, 1);
    cfg.blockDim = dim3(threads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, l);
}

template <typename TI, typename TO, bool WIDE, uint32_t MAX_ROWS>
cudaError_t launch_adjust(const AdjustLaunch<MAX_ROWS> &l, const Cut &cut, cudaStream_t stream) {
    return launch(adjust_logits_kernel<TI, TO, WIDE, MAX_ROWS>, l, l.a.tasks, NT, cut.smem, stream);
}

template <typename TI, typename TO, uint32_t MAX_ROWS>
cudaError_t adjust_by_cut(const AdjustLaunch<MAX_ROWS> &l, bool wide, const Cut &cut, cudaStream_t stream) {
    return wide ? launch_adjust<TI, TO, true, MAX_ROWS>(l, cut, stream) : launch_adjust<TI, TO, false, MAX_ROWS>(l, cut, stream);
}

// The rows [row0, row0 + rows) of a call, their penalties and slots in the launch's arguments.
template <uint32_t MAX_ROWS>
cudaError_t adjust_rows(const AdjustArgs &a, const lily_adjust_args_t &g, uint32_t row0, uint32_t rows, bool wide,
                        const Cut &cut, cudaStream_t stream) {
    AdjustLaunch<MAX_ROWS> l;
    l.a = a;
    l.a.row0 = row0, l.a.rows = rows, l.a.tasks = rows * cut.slices;
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
    using B = __nv_bfloat16;
    return g.logits_dtype == LILY_F32 ? adjust_by_cut<float, float>(l, wide, cut, stream)
           : g.out_dtype == LILY_F32  ? adjust_by_cut<B, float>(l, wide, cut, stream)
                                      : adjust_by_cut<B, B>(l, wide, cut, stream);
}

cudaError_t mask_rows(const AdjustArgs &a, const lily_adjust_args_t &g, uint32_t row0, uint32_t rows, bool wide, const Cut &cut,
                      cudaStream_t stream) {
    AdjustLaunch<1> l;
    l.a = a;
    l.a.row0 = row0, l.a.rows = rows, l.a.tasks = rows * cut.slices;
    using B = __nv_bfloat16;
    const auto go = [&](auto narrow_kernel, auto wide_kernel) {
        return launch(wide ? wide_kernel : narrow_kernel, l, l.a.tasks, MASK_NT, cut.smem, stream);
    };
    return g.logits_dtype == LILY_F32 ? go(mask_logits_kernel<float, float, false>, mask_logits_kernel<float, float, true>)
           : g.out_dtype == LILY_F32  ? go(mask_logits_kernel<B, float, false>, mask_logits_kernel<B, float, true>)
                                      : go(mask_logits_kernel<B, B, false>, mask_logits_kernel<B, B, true>);
}

constexpr uint32_t ROWS_FEW = 16, ROWS_MANY = 256;

// The variants that a call chooses from.
template <typename TI, typename TO, bool WIDE>
cudaError_t load_adjusts() {
    for (const cudaError_t e : {load_kernel(mask_logits_kernel<TI, TO, WIDE>), load_kernel(adjust_logits_kernel<TI, TO, WIDE, 1>, MOST_SMEM),
                                load_kernel(adjust_logits_kernel<TI, TO, WIDE, ROWS_FEW>, MOST_SMEM),
                                load_kernel(adjust_logits_kernel<TI, TO, WIDE, ROWS_MANY>, MOST_SMEM)}) {
        if (e != cudaSuccess) {
            return e;
        }
    }
    return cudaSuccess;
}

}  // namespace

cudaError_t lily_host::adjust_ready() {
    static std::atomic<uint64_t> seen{0};
    return once_per_device(seen, [] {
        using B = __nv_bfloat16;
        for (const cudaError_t e : {load_adjusts<float, float, false>(), load_adjusts<float, float, true>(), load_adjusts<B, float, false>(),
                                    load_adjusts<B, float, true>(), load_adjusts<B, B, false>(), load_adjusts<B, B, true>()}) {
            if (e != cudaSuccess) {
                return e;
            }
        }
        return cudaSuccess;
    });
}

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
    for (const void *words : {(const void *)g.history_ids, (const void *)g.history_len, (const void *)g.bias_ids, (const void *)g.bias_vals,
                              (const void *)g.bias_len, (const void *)g.ban_ids, (const void *)g.ban_len, (const void *)g.mask,
                              (const void *)g.mask_rows, (const void *)g.out_status}) {
        if (reinterpret_cast<uintptr_t>(words) % 4u) {
            return fail(h, LILY_ERR_ARG, "a list, a mask or a status is not aligned to its words");
        }
    }
    if (g.params_on_device && reinterpret_cast<uintptr_t>(g.params) % alignof(lily_sampling_params_t)) {
        return fail(h, LILY_ERR_ARG, "params are not aligned");
    }
    if ((uint64_t)g.first_id + h->vocab > 0xFFFFFFFFull) {
        return fail(h, LILY_ERR_ARG, "first_id + vocab overflows an id");
    }
    if (g.mask != nullptr && (g.mask_ld * 32u < (uint64_t)g.first_id + h->vocab || g.masks == 0u ||
                              (g.mask_rows == nullptr && g.masks < g.rows))) {
        return fail(h, LILY_ERR_ARG, "masks of at least first_id + vocab bits, one per row if mask_rows is NULL");
    }
    if (g.mask != nullptr && (uint64_t)g.first_id + h->vocab > 0x7FFFFFFFull) {
        return fail(h, LILY_ERR_CAPACITY, "masks take ids up to 2^31 - 1");
    }
    if (g.mask == nullptr && g.mask_rows != nullptr) {
        return fail(h, LILY_ERR_ARG, "mask_rows without mask");
    }
    if (g.count_slots != nullptr && (h->counts_table == nullptr || g.first_id != 0u)) {
        return fail(h, LILY_ERR_ARG, "count_slots needs LILY_FLAG_COUNTS_TABLE and first_id 0");
    }
    bool penalties = g.params != nullptr && g.params_on_device;
    for (uint32_t r = 0; r < g.rows; ++r) {
        if (g.params != nullptr && !g.params_on_device) {
            if (!params_ok(g.params[r])) {
                char buf[64];
                std::snprintf(buf, sizeof buf, "row %u: invalid sampling parameters", r);
                return fail(h, LILY_ERR_PARAMS, buf);
            }
            penalties = penalties || g.params[r].frequency_penalty != 0.0f || g.params[r].presence_penalty != 0.0f || g.params[r].repetition_penalty != 1.0f;
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

    // Rows of both buffers miss the boundaries of eight logits alike (or not at all).
    const bool wide = reinterpret_cast<uintptr_t>(g.logits) / in_size % 8u == reinterpret_cast<uintptr_t>(g.out) / out_size % 8u &&
                      (g.rows == 1u || g.logits_ld % 8u == g.out_ld % 8u);
    const bool lists = history || g.bias_ids != nullptr || (penalties && g.count_slots != nullptr);
    const bool keeps = g.mask != nullptr || g.ban_ids != nullptr || g.bias_ids != nullptr;
    a.history_ids = history ? g.history_ids : nullptr;
    const uint64_t most_times = std::min<uint64_t>(g.history_ld, h->max_history);  // that a list has an id
    const auto slice_of = [&](uint32_t count) { return ((h->vocab + count - 1u) / count + 255u) & ~255u; };
    const auto lay_out = [&](uint32_t slice) -> size_t {  // a block's shared memory
        const uint32_t words = slice / 32u + 8u;
        a.direct = slice + 8u <= 2u * WINDOW ? 1u : slice + 32u <= 4u * WINDOW && most_times <= 65535u ? 2u : 0u;
        a.seen_at = keeps ? words : 0u;
        a.before_at = a.seen_at + (history && !a.direct ? words : 0u);
        return (a.before_at + (history && !a.direct ? words : 0u)) * 4u;
    };
    // Slices: as many as fill the device with two blocks an SM, of LEAST_SLICE logits at least.
    const uint32_t resident = 2u * (uint32_t)h->sm_count;
    Cut cut = {std::max(1u, std::min(resident / g.rows, (h->vocab + LEAST_SLICE - 1u) / LEAST_SLICE)), 0u};
    while (lay_out(slice_of(cut.slices)) > (lists ? MOST_SMEM : 47u * 1024u)) {
        ++cut.slices;
    }
    a.slice_len = slice_of(cut.slices);
    cut.slices = (h->vocab + a.slice_len - 1u) / a.slice_len;  // (rounded up, they may be fewer)
    cut.smem = lay_out(a.slice_len);

    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    const bool plain = (g.params == nullptr || g.params_on_device) && g.count_slots == nullptr;
    const uint32_t step = !lists || plain ? 0x7FFFFFFFu / cut.slices : ROWS_MANY;
    for (uint32_t r = 0; r < g.rows; r += step) {
        const uint32_t rows = std::min(step, g.rows - r);
        if (!lists) {
            CU(h, mask_rows(a, g, r, rows, wide, cut, stream));
        } else if (plain) {
            CU(h, adjust_rows<1>(a, g, r, rows, wide, cut, stream));
        } else if (rows <= ROWS_FEW) {
            CU(h, adjust_rows<ROWS_FEW>(a, g, r, rows, wide, cut, stream));
        } else {
            CU(h, adjust_rows<ROWS_MANY>(a, g, r, rows, wide, cut, stream));
        }
    }
    return LILY_OK;
}
