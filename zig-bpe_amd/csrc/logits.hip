// The operators between a model's logits and its tokens (include/zbpe.h): grammar masks over the vocabulary, penalties /
// biases / masks on logits and their gradient, the draw of a token, log-probabilities and their gradient.
#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include <exception>
#include <new>
#include <utility>

#include "../../include/zbpe.h"
#include "logits.hpp"
#include "vocab.hpp"
#include "wave.hpp"

namespace zbpe {

static thread_local char g_message[512] = "";
const char *thread_message() { return g_message[0] ? g_message : nullptr; }
void forget_thread_message() { g_message[0] = 0; }

__attribute__((format(printf, 2, 3))) static zbpe_status refuse(zbpe_status s, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_message, sizeof g_message, fmt, ap);
    va_end(ap);
    return s;
}

// The same in every lane of a wave: in scalar registers.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }
__device__ __forceinline__ float uniform(float x) { return __uint_as_float(uniform(__float_as_uint(x))); }
__device__ __forceinline__ uint64_t uniform(uint64_t x) {
    return (uint64_t)uniform((uint32_t)(x >> 32)) << 32 | uniform((uint32_t)x);
}
__device__ __forceinline__ double uniform(double x) { return __longlong_as_double((int64_t)uniform((uint64_t)__double_as_longlong(x))); }

// ---- rows ---------------------------------------------------------------------------------------------------------------

// One matrix of a launch: where row r starts.
struct Rows {
    char *data;
    int64_t outer, inner;  // strides, in elements
};
template <class T>
__device__ __forceinline__ T *row_of(const Rows &m, int64_t r, int64_t per) {
    // (the common case of one stride: no division)
    const int64_t at = m.outer == per * m.inner ? r * m.inner : (r / per) * m.outer + (r % per) * m.inner;
    return (T *)m.data + at;
}

// A row's place in both levels, for walks over consecutive rows: one division for all of them.
struct RowAt {
    int64_t outer, inner;
    __device__ __forceinline__ RowAt(int64_t r, int64_t per) : outer((int64_t)uniform((uint64_t)(r / per))), inner((int64_t)uniform((uint64_t)(r % per))) {}
    __device__ __forceinline__ void next(int64_t per) {
        if (++inner == per) {
            inner = 0;
            outer++;
        }
    }
    template <class T, int SIZE = sizeof(T)>
    __device__ __forceinline__ T *of(const Rows &m) const { return (T *)(m.data + (outer * m.outer + inner * m.inner) * SIZE); }
};

using f16 = _Float16;
using bf16 = __bf16;

// The same number, worked with anew: what is computed from it for the ends of rows is not kept in registers through whole loops.
__device__ __forceinline__ int afresh(int x) {
    asm volatile("" : "+s"(x));
    return x;
}
__device__ __forceinline__ uint32_t afresh(uint32_t x) {  // different in every lane
    asm volatile("" : "+v"(x));
    return x;
}

// 16 bytes of elements. Rows may start at any element (an odd number of columns): the copies below are 16-byte loads and
// stores at the element's alignment, which global memory allows.
template <class T>
struct Pack {
    static constexpr int N = 16 / sizeof(T);
    T v[N];
};
template <class T>
__device__ __forceinline__ Pack<T> load_pack(const T *p) {
    Pack<T> x;
    __builtin_memcpy(&x, p, sizeof x);
    return x;
}
// N elements as they are in memory, two of 16 bits in a register; 0 past the row's end
template <class T, int N>
struct Raw {
    uint32_t word[N * sizeof(T) / 4];
    __device__ __forceinline__ void load(const T *row, int col, int cols) {
        if (col + N <= cols) {
            __builtin_memcpy(word, (const char *)row + (uint32_t)col * (uint32_t)sizeof(T), sizeof word);
        } else {
            const int left = afresh(cols) - col;
#pragma unroll
            for (int i = 0; i < (int)(N * sizeof(T) / 4); i++) word[i] = 0;
#pragma unroll
            for (int e = 0; e < N; e++) {
                uint32_t x = 0;
                if (e < left) __builtin_memcpy(&x, (const char *)row + ((uint32_t)col + e) * (uint32_t)sizeof(T), sizeof(T));
                if (sizeof(T) == 4) word[e] = x;
                else word[e / 2] |= x << (16 * (e & 1));
            }
        }
    }
    __device__ __forceinline__ float get(int e) const {
        const uint32_t x = sizeof(T) == 4 ? word[e] : e & 1 ? word[e / 2] >> 16 : word[e / 2] & 0xffff;
        T v;
        __builtin_memcpy(&v, &x, sizeof(T));
        return (float)v;
    }
};

// N consecutive elements as floats; those past `cols` become `fill`.
template <class T, int N>
__device__ __forceinline__ void load_floats(const T *row, int col, int cols, float fill, float *z) {
    static_assert(N % Pack<T>::N == 0, "whole packs");
    if (col + N <= cols) {
#pragma unroll
        for (int k = 0; k < N; k += Pack<T>::N) {
            const Pack<T> x = load_pack(row + col + k);
#pragma unroll
            for (int e = 0; e < Pack<T>::N; e++) z[k + e] = (float)x.v[e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < N; e++) z[e] = col + e < cols ? (float)row[col + e] : fill;
    }
}
template <class T, int N>
__device__ __forceinline__ void store_floats(T *row, int col, int cols, const float *z) {
    if (col + N <= cols) {
        T x[N];
#pragma unroll
        for (int e = 0; e < N; e++) x[e] = (T)z[e];
        __builtin_memcpy((char *)row + (uint32_t)col * (uint32_t)sizeof(T), x, sizeof x);
    } else {
        const int left = afresh(cols) - col;
#pragma unroll
        for (int e = 0; e < N; e++)
            if (e < left) row[col + e] = (T)z[e];
    }
}

constexpr float INF = __builtin_huge_valf();

// ---- wave and workgroup sums --------------------------------------------------------------------------------------------

__device__ __forceinline__ float wave_max(float x) {
    for (int d = 32; d; d >>= 1) x = fmaxf(x, __shfl_xor(x, d));
    return x;
}
__device__ __forceinline__ float wave_sum(float x) {
    for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
    return x;
}
__device__ __forceinline__ uint64_t wave_sum(uint64_t x) {
    for (int d = 32; d; d >>= 1) x += __shfl_xor((unsigned long long)x, d);
    return x;
}
__device__ __forceinline__ uint64_t wave_scan(uint64_t x) {  // inclusive
    const int lane = threadIdx.x & 63;
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t y = __shfl_up((unsigned long long)x, d);
        if (lane >= d) x += y;
    }
    return x;
}

// ---- grammar masks ------------------------------------------------------------------------------------------------------

struct Automaton {
    const uint32_t *offsets;
    const uint8_t *bytes;
    const int32_t *next;
    const uint8_t *accepting;
    const void *index;
    int vocab, end, n;
};

__device__ __forceinline__ bool inside(const Automaton &g, int s) { return (uint32_t)s < (uint32_t)g.n; }

// The state after bytes [at, to) from s; -1 once it is outside the automaton.
__device__ __forceinline__ int walk(const Automaton &g, int s, uint32_t at, uint32_t to) {
    while (at < to && inside(g, s)) s = g.next[(int64_t)s * 256 + g.bytes[at++]];
    return inside(g, s) ? s : -1;
}

// One workgroup makes one state's bits of some slices of ids. Most tokens need no walk:
//   - A slice's tokens come in the order of their bytes (vocab.hpp), so 64 neighbours begin alike; where the state refuses all of
//     their first bytes, they are not even read.
//   - Most bytes of an answer leave the state as it is (the inside of a string, a number's digits). A token carries the set of its
//     bytes' classes; when no class in it holds a byte that changes the state, the token is allowed.
//   - Of the others most end at their second byte.
// Each wave queues what is left and walks it 64 at a time. The rows of the automaton that such walks need most, the state's own
// and up to three that follow it (seven: 3 % slower, since every state pays for them), are in shared memory, their entries
// replaced by the places of these rows (0 .. ROWS - 1, then REFUSED, then all other states). The bits return to the order of ids in
// shared memory. 2048 states x 65535 tokens in 172 us (a walk for each pair: 728), 600 x 32000 in 40; the 19 MB in and out would
// take 4. What bounds it: the instructions of classifying and walking (vector instructions issue in 59 % of busy cycles) and, in
// the rest, the latency of a state's rows, which every workgroup of a state prepares anew.
template <int NT>
__global__ __launch_bounds__(NT) void grammar_masks_kernel(Automaton g, const int32_t *states, int64_t rows, uint32_t *masks, int slices, int per) {
    constexpr int ROWS = 4, REFUSED = ROWS, SLICES = ZBPE_MAX_VOCAB / INDEX_SLICE, SLICE_WORDS = INDEX_SLICE / 32;
    __shared__ int next[ROWS + 1][256];  // the last row: once refused, always refused
    __shared__ int place[ROWS];  // the states of these rows
    __shared__ uint32_t live[8], turns[2][4];  // the bytes that the state takes; the classes with a byte that changes it
    __shared__ uint32_t bits[SLICES * SLICE_WORDS];
    __shared__ uint16_t list[SLICES * INDEX_SLICE / 64];
    __shared__ uint16_t queues[NT / 64][128];
    __shared__ int listed;
    const int t = threadIdx.x, lane = t & 63, wave = (int)uniform((uint32_t)t >> 6), words = (g.vocab + 31) / 32;
    const int parts = (slices + per - 1) / per;
    const IndexView index(g.index, g.vocab);
    uint16_t *queue = queues[wave];
    for (int64_t w = blockIdx.x; w < rows * parts; w += gridDim.x) {
        const int64_t r = w / parts;
        const int first_slice = (int)(w % parts) * per, last_slice = first_slice + per < slices ? first_slice + per : slices;
        const int first_word = first_slice * SLICE_WORDS, last_word = min(last_slice * SLICE_WORDS, words);
        const int first_group = first_slice * (INDEX_SLICE / 64), last_group = min(last_slice * (INDEX_SLICE / 64), (g.vocab + 63) / 64);
        const int s0 = states ? states[r] : (int)r;
        const bool known = inside(g, s0);
        __syncthreads();
        if (t < 256) {
            const int to = known ? g.next[(int64_t)s0 * 256 + t] : -1;
            const bool on = inside(g, to);
            next[0][t] = on ? to : -1;
            const uint64_t b = __ballot(on);
            if (lane == 0) live[t >> 5] = (uint32_t)b;
            if (lane == 32) live[t >> 5] = (uint32_t)(b >> 32);
            const int c = byte_class(t);
            const uint32_t low = wave_or_u32(to != s0 && c < 32 ? 1u << c : 0u), high = wave_or_u32(to != s0 && c >= 32 ? 1u << (c - 32) : 0u);
            if (lane == 0) {
                turns[0][wave] = low;
                turns[1][wave] = high;
            }
        }
        for (int i = t; i < last_word - first_word; i += NT) {
            const bool ends = g.end >= 0 && g.end / 32 == first_word + i && known && g.accepting && g.accepting[s0];
            bits[i] = ends ? 1u << (g.end & 31) : 0u;
        }
        if (t == 0) listed = 0;
        __syncthreads();
        for (int i = first_group + t; i < last_group; i += NT) {
            const IndexBounds x = index.bounds[i];
            uint32_t any = 0;
            for (int i = x.lo >> 5; i <= x.hi >> 5; i++) {
                uint32_t m = live[i];
                if (i == x.lo >> 5) m &= ~0u << (x.lo & 31);
                if (i == x.hi >> 5) m &= ~0u >> (31 - (x.hi & 31));
                any |= m;
            }
            if (any) list[atomicAdd(&listed, 1)] = (uint16_t)i;  // (in any order: each group has bits of its own)
        }
        if (wave == NT / 64 - 1) {  // the first states that follow, each once
            int to[4];
#pragma unroll
            for (int i = 0; i < 4; i++) to[i] = next[0][i * 64 + lane];
            int chosen = s0;
            for (int k = 0; k < ROWS; k++) {
                int mine = -1;
#pragma unroll
                for (int i = 3; i >= 0; i--) {
                    if (to[i] == chosen) to[i] = -1;
                    if (to[i] >= 0) mine = to[i];
                }
                if (lane == 0) place[k] = chosen;
                const uint64_t b = __ballot(mine >= 0);
                chosen = b ? (int)lane_bcast((uint32_t)mine, __ffsll((unsigned long long)b) - 1) : -1;
            }
        }
        __syncthreads();
        for (int i = t; i < (ROWS + 1) * 256; i += NT) {
            const int s = i < ROWS * 256 ? place[i >> 8] : -1;
            int to = i < 256 ? next[0][i] : s >= 0 && known ? g.next[(int64_t)s * 256 + (i & 255)] : -1;
            if (!inside(g, to)) to = REFUSED;
            else {
                int at = to + ROWS + 1;
#pragma unroll
                for (int k = ROWS - 1; k >= 0; k--)
                    if (to == place[k]) at = k;
                to = at;
            }
            next[i >> 8][i & 255] = to;
        }
        __syncthreads();
        const uint32_t turns_low = turns[0][0] | turns[0][1] | turns[0][2] | turns[0][3];
        const uint32_t turns_high = turns[1][0] | turns[1][1] | turns[1][2] | turns[1][3];

        auto allow = [&](int id) { atomicOr(&bits[(id >> 5) - first_word], 1u << (id & 31)); };
        auto walk_queued = [&](int i) {
            const int at = queue[i];
            const IndexHead x = index.heads[at];
            const IndexTail y = index.tails[at];
            const int id = at / INDEX_SLICE * INDEX_SLICE + x.id(), length = x.length();
            int s = 0;
#pragma unroll
            for (int j = 0; j < INDEX_BYTES; j++) {
                if (j % 3 == 0 && !__any(s != REFUSED && j < length)) break;
                const int b = j < INDEX_HEAD ? x.byte(j) : y.byte(j - INDEX_HEAD);
                int to = next[min(s, REFUSED)][b];
                if (s > REFUSED && j < length) {
                    to = g.next[(int64_t)(s - ROWS - 1) * 256 + b];
                    to = inside(g, to) ? to == s0 ? 0 : to + ROWS + 1 : REFUSED;
                }
                s = j < length ? to : s;
            }
            if (length > INDEX_BYTES && s != REFUSED) {
                s = walk(g, s < ROWS ? place[s] : s - ROWS - 1, g.offsets[id] + INDEX_BYTES, g.offsets[id + 1]);
                if (s < 0) s = REFUSED;
            }
            if (s != REFUSED) allow(id);
        };

        const int n = (int)uniform((uint32_t)listed);
        auto group = [&](int i) { return (int)uniform((uint32_t)list[i]) * 64; };
        int queued = 0, first = 0;
        IndexHead ahead{};
        if (wave < n) ahead = index.heads[(first = group(wave)) + lane];
        for (int i = wave; i < n; i += NT / 64) {
            const IndexHead x = ahead;
            const int from = first;
            if (i + NT / 64 < n) ahead = index.heads[(first = group(i + NT / 64)) + lane];
            const int id = from / INDEX_SLICE * INDEX_SLICE + x.id(), length = x.length();
            const bool asked = length && id != g.end;
            bool on = asked && !((x.classes[0] & turns_low) | (x.classes[1] & turns_high)), open = false;
            if (__any(asked && !on)) {
                const int s = next[0][x.byte(0)];
                const bool fits = length == 1 ? s != REFUSED : s > REFUSED || next[min(s, REFUSED)][x.byte(1)] != REFUSED;
                const bool ends = length == 1 || (length == 2 && s < REFUSED);
                open = asked && !on && fits && !ends;
                on = on || (asked && fits && ends);
            }
            if (on) allow(id);
            const uint64_t b = __ballot(open);
            if (open) queue[queued + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, 0))] = (uint16_t)(from + lane);
            queued += __popcll(b);
            if (queued >= 64) {
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                queued -= 64;
                walk_queued(queued + lane);
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (lane < queued) walk_queued(lane);
        __syncthreads();
        for (int i = t; i < last_word - first_word; i += NT) masks[r * words + first_word + i] = bits[i];
    }
}

__global__ __launch_bounds__(256) void grammar_advance_kernel(Automaton g, const int32_t *states, const int32_t *tokens, int64_t rows, int32_t *out) {
    for (int64_t r = blockIdx.x * 256ll + threadIdx.x; r < rows; r += gridDim.x * 256ll) {
        const int s = states[r], v = tokens[r];
        int to = -1;
        if (inside(g, s)) {
            if (v < 0) to = s;
            else if (v >= g.vocab) to = -1;
            else if (v == g.end) to = g.accepting && g.accepting[s] ? s : -1;
            else if (g.offsets[v] < g.offsets[v + 1]) to = walk(g, s, g.offsets[v], g.offsets[v + 1]);
        }
        out[r] = to;
    }
}

// ---- penalties, biases and masks ----------------------------------------------------------------------------------------

// A workgroup takes a slice of columns over a run of rows, 32 bytes of logits a thread. What a row needs from memory is on its
// way while the row before it is worked on. The row's history is counted in shared memory: a bit for each column that is in it
// (the bits of one load's columns in one byte, which is 0 for most loads) and how often behind the prompt. Whoever uses a bit
// or a count clears it. 4096 rows of 32000 bf16, up to 500 tokens of history each, in 149 us (0.52 GB, 3.5 TB/s; a copy
// reaches 4.9), the gradient in 172. What bounds it: memory, with vector instructions in 55 % of busy cycles (the gradient: 41, and a
// scattered load for each place of the history). 256 rows with histories up to 2000 take 30 us: a run is two rows, and each of
// four slices counts all of a row's history, what lies behind the first 512 tokens within the row's turn.
constexpr int ADJUST_THREADS = 512, ADJUST_PACKS = 2, ADJUST_RUN = 32;
constexpr int ADJUST_GROUPS = 2;  // on a CU at a time: 4 waves on a SIMD leave 128 registers to a thread
template <class T>
constexpr int ADJUST_SLICE = ADJUST_THREADS * ADJUST_PACKS * Pack<T>::N;

struct Adjust {
    Rows logits, out, history;
    int64_t rows, inner, mask_rows, runs;
    int cols, slices, run, words, n_biases, wide_ids;
    int64_t history_len;
    const int32_t *lengths, *prompt_lengths, *bias_tokens, *states;
    const float *repetition, *presence, *frequency, *bias, *bias_values;
    const uint32_t *masks;
};

// What is known of each row of a run.
struct AdjustRows {
    const uint32_t *mask[ADJUST_RUN];  // null: everything is masked
    int length[ADJUST_RUN], prompt[ADJUST_RUN];
    float theta[ADJUST_RUN], presence[ADJUST_RUN], frequency[ADJUST_RUN];
    __device__ __forceinline__ void load(const Adjust &a, int64_t first, int64_t last) {
        const int i = threadIdx.x;
        const int64_t r = first + i;
        __syncthreads();
        if (r < last && i < ADJUST_RUN) {
            const int64_t m = a.states ? a.states[r] : a.mask_rows == 1 ? 0 : r;
            mask[i] = a.masks && m >= 0 && m < a.mask_rows ? a.masks + m * a.words : nullptr;
            const int n = a.lengths ? a.lengths[r] : (int)a.history_len;
            length[i] = n < 0 ? 0 : n > a.history_len ? (int)a.history_len : n;
            prompt[i] = a.prompt_lengths ? a.prompt_lengths[r] : 0;
            theta[i] = a.repetition ? a.repetition[r] : 1.0f;
            presence[i] = a.presence ? a.presence[r] : 0.0f;
            frequency[i] = a.frequency ? a.frequency[r] : 0.0f;
        }
        __syncthreads();
    }
};

// A token of a row's history, as it comes from memory: that at the thread's place, if no other is named
struct Recent {
    uint32_t low, high;
    __device__ __forceinline__ void load(const Adjust &a, const RowAt &at, uint32_t place = threadIdx.x) {
        low = high = 0;
        if ((int64_t)place >= a.history_len) return;
        const char *ids = a.wide_ids ? at.of<char, 8>(a.history) : at.of<char, 4>(a.history);
        const uint64_t from = (uint64_t)place << (2 + a.wide_ids);
        low = *(const uint32_t *)(ids + from);
        high = *(const uint32_t *)(ids + (from + 4 * a.wide_ids));
    }
    __device__ __forceinline__ int64_t get(int wide) const { return wide ? (int64_t)((uint64_t)high << 32 | low) : (int64_t)(int32_t)low; }
};

// f(place, token) for a row's n tokens of history, over the workgroup's threads
template <class F>
__device__ __forceinline__ void each_history(const Adjust &a, const Recent &recent, int n, const RowAt &at, F f) {
    if ((int)threadIdx.x < n) f((int)threadIdx.x, recent.get(a.wide_ids));
    constexpr int AHEAD = 4;
    for (uint32_t i = afresh(threadIdx.x) + ADJUST_THREADS; i < (uint32_t)n; i += AHEAD * ADJUST_THREADS) {
        Recent x[AHEAD];
#pragma unroll
        for (int q = 0; q < AHEAD; q++) x[q].load(a, at, i + q * ADJUST_THREADS);
#pragma unroll
        for (int q = 0; q < AHEAD; q++)
            if (i + q * ADJUST_THREADS < (uint32_t)n) f((int)(i + q * ADJUST_THREADS), x[q].get(a.wide_ids));
    }
}

// One bit a column: those of the N columns that one load brings are the low bits of one byte.
template <int N>
struct Flags {
    static constexpr int WORDS = ADJUST_THREADS * ADJUST_PACKS / 4;
    uint32_t word[WORDS];
    __device__ __forceinline__ void set(uint32_t k) { atomicOr(&word[k / (4 * N)], 1u << (k / N % 4 * 8 + k % N)); }
    // the bits of columns k .. k + N, cleared
    __device__ __forceinline__ uint32_t take(int k) {
        uint8_t *at = (uint8_t *)word + k / N;
        const uint32_t x = *at;
        if (x) *at = 0;
        return x;
    }
};

// x[e] of values that stay in registers: by bits, since choices between elements would be turned into an array in memory
template <int N>
__device__ __forceinline__ float pick(const float *x, int e) {
    uint32_t v = 0;
#pragma unroll
    for (int i = 0; i < N; i++) v |= __float_as_uint(x[i]) & (i == e ? ~0u : 0u);
    return __uint_as_float(v);
}
template <int N>
__device__ __forceinline__ void put(float *x, int e, float v) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        const uint32_t m = i == e ? ~0u : 0u;
        x[i] = __uint_as_float((__float_as_uint(x[i]) & ~m) | (__float_as_uint(v) & m));
    }
}

// The rows and columns of one piece of work of a launch.
struct AdjustPart {
    int64_t first, last;  // rows
    int base, width;      // columns
};
template <class T>
__device__ __forceinline__ AdjustPart part_of(const Adjust &a, int64_t w) {
    AdjustPart p;
    const int64_t run = (int64_t)uniform((uint64_t)(w / a.slices));
    p.first = run * a.run;
    p.last = p.first + a.run < a.rows ? p.first + a.run : a.rows;
    p.base = (int)(w - run * a.slices) * ADJUST_SLICE<T>;
    p.width = a.cols - p.base < ADJUST_SLICE<T> ? a.cols - p.base : ADJUST_SLICE<T>;
    return p;
}

// The word of a row's mask that holds column col's bit and those of its load (their number divides 32).
__device__ __forceinline__ uint32_t mask_word(const Adjust &a, const uint32_t *mask, int col) {
    return !a.masks ? ~0u : mask && col < a.cols ? mask[col >> 5] : 0u;
}

template <class Ti, class To>
__global__ __launch_bounds__(ADJUST_THREADS, 2 * ADJUST_GROUPS) void adjust_kernel(Adjust a) {
#pragma clang fp contract(off)
    constexpr int N = Pack<Ti>::N, C = ADJUST_PACKS, NT = ADJUST_THREADS;
    __shared__ uint32_t counts[ADJUST_SLICE<Ti>];
    __shared__ AdjustRows known;
    __shared__ Flags<N> seen, special;  // in the history; with a bias of the row's own
    __shared__ int bias_token[ZBPE_MAX_BIASES];
    __shared__ float bias_value[ZBPE_MAX_BIASES];
    const int t = threadIdx.x;
    const bool past = a.history.data != nullptr, biased = a.n_biases > 0;
    if (past)
        for (int i = t; i < ADJUST_SLICE<Ti>; i += NT) counts[i] = 0;
    for (int i = t; i < Flags<N>::WORDS; i += NT) seen.word[i] = special.word[i] = 0;
    for (int64_t w = blockIdx.x; w < a.runs * a.slices; w += gridDim.x) {
        const AdjustPart part = part_of<Ti>(a, w);
        Raw<Ti, N> next[C];
        Raw<float, N> bias[C];
        RowAt at(part.first, a.inner), ahead = at;
        Recent recent{};
        if (past) recent.load(a, at);
        int own_token = -1;  // entry t of the next row's biases
        float own_value = 0.0f;
        if (t < a.n_biases) {
            own_token = a.bias_tokens[part.first * a.n_biases + t];
            own_value = a.bias_values[part.first * a.n_biases + t];
        }
        uint32_t masked[C];  // the next row's
        known.load(a, part.first, part.last);
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int col = part.base + (c * NT + t) * N;
            next[c].load(at.of<Ti>(a.logits), col, a.cols);
            masked[c] = mask_word(a, known.mask[0], col);
            if (a.bias) bias[c].load(a.bias, col, a.cols);
            else
#pragma unroll
                for (int e = 0; e < N; e++) bias[c].word[e] = 0x80000000u;  // -0: what adds nothing
        }
        for (int64_t r = part.first; r < part.last; r++, at = ahead) {
            ahead.next(a.inner);
            const int i = (int)(r - part.first);
            const bool more = r + 1 < part.last;
            Raw<Ti, N> z[C];
            uint32_t allowed[C];
#pragma unroll
            for (int c = 0; c < C; c++) {
                const int col = part.base + (c * NT + t) * N;
                z[c] = next[c];
                allowed[c] = masked[c] >> (col & 31);
                if (more) {
                    next[c].load(ahead.of<Ti>(a.logits), col, a.cols);
                    masked[c] = mask_word(a, known.mask[i + 1], col);
                }
            }
            const Recent tokens = recent;
            if (past && more) recent.load(a, ahead);
            const int token = own_token;
            const float value = own_value;
            if (more && t < a.n_biases) {
                own_token = a.bias_tokens[(r + 1) * a.n_biases + t];
                own_value = a.bias_values[(r + 1) * a.n_biases + t];
            }
            if (past || biased) {
                __syncthreads();  // what the last row used is clear
                if (past) {
                    const int prompt = known.prompt[i];
                    each_history(a, tokens, known.length[i], at, [&](int i, int64_t id) {
                        const uint64_t k = (uint64_t)(id - part.base);
                        if (k >= (uint64_t)part.width) return;
                        seen.set((uint32_t)k);
                        if (i >= prompt) atomicAdd(&counts[k], 1u);
                    });
                }
                for (int j = t; j < a.n_biases; j += NT) {
                    const int id = j < NT ? token : a.bias_tokens[r * a.n_biases + j];
                    bias_token[j] = id;
                    bias_value[j] = j < NT ? value : a.bias_values[r * a.n_biases + j];
                    const uint32_t k = (uint32_t)id - (uint32_t)part.base;
                    if (k < (uint32_t)part.width) special.set(k);
                }
                __syncthreads();
            }
            To *out = at.of<To>(a.out);
#pragma unroll
            for (int c = 0; c < C; c++) {
                const int k = (c * NT + t) * N, col = part.base + k;
                if (col >= a.cols) continue;
                float y[N];
#pragma unroll
                for (int e = 0; e < N; e++) y[e] = z[c].get(e);
                if (past) {
                    uint32_t old = seen.take(k);
                    if (old) {
                        const float theta = known.theta[i], presence = known.presence[i], frequency = known.frequency[i];
#pragma unroll 1
                        for (; old; old &= old - 1) {
                            const int e = __ffs(old) - 1;
                            float x = pick<N>(y, e);
                            x = x > 0.0f ? x / theta : x * theta;
                            const uint32_t count = counts[k + e];
                            if (count) {
                                counts[k + e] = 0;
                                x = x - frequency * (float)count;
                                x = x - presence;
                            }
                            put<N>(y, e, x);
                        }
                    }
                }
#pragma unroll
                for (int e = 0; e < N; e++) y[e] = y[e] + bias[c].get(e);
                if (biased && special.take(k)) {
                    // all of the row's entries in their order; those of one column are summed first
                    float sum[N];
#pragma unroll
                    for (int e = 0; e < N; e++) sum[e] = -0.0f;
#pragma unroll 4
                    for (int j = 0; j < a.n_biases; j++) {
                        const uint32_t place = (uint32_t)bias_token[j] - (uint32_t)col;
                        const float value = bias_value[j];
#pragma unroll
                        for (int e = 0; e < N; e++) sum[e] += place == (uint32_t)e ? value : -0.0f;
                    }
#pragma unroll
                    for (int e = 0; e < N; e++) y[e] = y[e] + sum[e];
                }
#pragma unroll
                for (int e = 0; e < N; e++) y[e] = (allowed[c] >> e) & 1 ? y[e] : -INF;
                store_floats<To, N>(out, col, a.cols, y);
            }
        }
    }
}

// dz = dy * slope, masked; the sum over rows of the masked dy for the shared bias: a workgroup keeps its columns' sums in
// registers over its run of rows and leaves them in the workspace; a second kernel adds the runs up in their order.
struct AdjustGrad {
    Adjust a;  // a.out: the gradient of the output
    Rows grad_logits;
    float *grad_bias_values, *sums;
};

template <class Ti, class To>
__global__ __launch_bounds__(ADJUST_THREADS, 2 * ADJUST_GROUPS) void adjust_grad_kernel(AdjustGrad g) {
    const Adjust &a = g.a;
    constexpr int N = Pack<Ti>::N, C = ADJUST_PACKS, NT = ADJUST_THREADS;
    __shared__ Flags<N> seen, positive;  // in the history; and with a logit above 0
    __shared__ AdjustRows known;
    const int t = threadIdx.x;
    const bool past = a.history.data != nullptr && g.grad_logits.data != nullptr;
    for (int i = t; i < Flags<N>::WORDS; i += NT) seen.word[i] = positive.word[i] = 0;
    for (int64_t w = blockIdx.x; w < a.runs * a.slices; w += gridDim.x) {
        const AdjustPart part = part_of<Ti>(a, w);
        Raw<To, N> next[C];
        float sum[C][N] = {};
        RowAt at(part.first, a.inner), ahead = at;
        // tokens are loaded two rows ahead, their logits one
        Recent recent{}, later{};
        float logit = 0.0f;
        auto logit_of = [&](const Recent &x, const RowAt &row) {
            const uint64_t k = (uint64_t)(x.get(a.wide_ids) - part.base);
            return (int64_t)t < a.history_len && k < (uint64_t)part.width ? (float)row.of<Ti>(a.logits)[part.base + (uint32_t)k] : 0.0f;
        };
        if (past) {
            recent.load(a, at);
            logit = logit_of(recent, at);
            RowAt second = at;
            second.next(a.inner);
            if (part.first + 1 < part.last) later.load(a, second);
        }
        uint32_t masked[C];  // the next row's
        known.load(a, part.first, part.last);
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int col = part.base + (c * NT + t) * N;
            next[c].load(at.of<To>(a.out), col, a.cols);
            masked[c] = mask_word(a, known.mask[0], col);
        }
        for (int64_t r = part.first; r < part.last; r++, at = ahead) {
            ahead.next(a.inner);
            const int i = (int)(r - part.first);
            const bool more = r + 1 < part.last;
            Raw<To, N> up[C];
            uint32_t allowed[C];
#pragma unroll
            for (int c = 0; c < C; c++) {
                const int col = part.base + (c * NT + t) * N;
                up[c] = next[c];
                allowed[c] = masked[c] >> (col & 31);
                if (more) {
                    next[c].load(ahead.of<To>(a.out), col, a.cols);
                    masked[c] = mask_word(a, known.mask[i + 1], col);
                }
            }
            const Recent tokens = recent;
            const float z = logit;
            if (past && more) {
                recent = later;
                logit = logit_of(recent, ahead);
                RowAt second = ahead;
                second.next(a.inner);
                if (r + 2 < part.last) later.load(a, second);
            }
            if (past) {
                __syncthreads();
                each_history(a, tokens, known.length[i], at, [&](int place, int64_t id) {
                    const uint64_t k = (uint64_t)(id - part.base);
                    if (k >= (uint64_t)part.width) return;
                    seen.set((uint32_t)k);
                    if ((place < NT ? z : (float)at.of<Ti>(a.logits)[id]) > 0.0f) positive.set((uint32_t)k);
                });
                __syncthreads();
            }
#pragma unroll
            for (int c = 0; c < C; c++) {
                const int k = (c * NT + t) * N, col = part.base + k;
                if (col >= a.cols) continue;
                float d[N];
#pragma unroll
                for (int e = 0; e < N; e++) {
                    d[e] = (allowed[c] >> e) & 1 ? up[c].get(e) : 0.0f;
                    sum[c][e] += d[e];
                }
                if (!g.grad_logits.data) continue;
                uint32_t old = past ? seen.take(k) : 0u;
                if (old) {
                    const float theta = known.theta[i];
                    const uint32_t above = positive.take(k);
#pragma unroll 1
                    for (; old; old &= old - 1) {
                        const int e = __ffs(old) - 1;
                        const float x = pick<N>(d, e);
                        put<N>(d, e, (above >> e) & 1 ? x / theta : x * theta);
                    }
                }
                store_floats<Ti, N>(at.of<Ti>(g.grad_logits), col, a.cols, d);
            }
        }
        if (g.grad_bias_values) {  // those of all rows at once, so that their loads wait together
            const int n = (int)(part.last - part.first) * a.n_biases;
            for (int q = t; q < n; q += NT) {
                const int i = q / a.n_biases;
                const int64_t r = part.first + i;
                const int32_t id = a.bias_tokens[part.first * a.n_biases + q];
                float d = 0.0f;
                if (id < 0 || id >= a.cols) {
                    if (part.base) continue;  // (no slice holds it: the first one writes its 0)
                } else {
                    if (id < part.base || id >= part.base + part.width) continue;
                    const uint32_t *mask = known.mask[i];
                    if (!a.masks || (mask && (mask[id >> 5] >> (id & 31)) & 1)) d = (float)row_of<To>(a.out, r, a.inner)[id];
                }
                g.grad_bias_values[part.first * a.n_biases + q] = d;
            }
        }
        if (g.sums)
#pragma unroll
            for (int c = 0; c < C; c++)
                store_floats<float, N>(g.sums + w / a.slices * a.cols, part.base + (c * NT + t) * N, a.cols, sum[c]);
    }
}

__global__ __launch_bounds__(1024) void adjust_bias_kernel(const float *sums, int64_t runs, int cols, float *grad_bias) {
    constexpr int PARTS = 16;
    const int col = blockIdx.x * 64 + (threadIdx.x & 63), part = threadIdx.x >> 6;
    __shared__ float other[PARTS][64];
    float s = 0.0f;
    if (col < cols)
#pragma unroll 4
        for (int64_t i = part; i < runs; i += PARTS) s += sums[i * cols + col];
    other[part][threadIdx.x & 63] = s;
    __syncthreads();
    if (part || col >= cols) return;
    for (int i = 1; i < PARTS; i++) s += other[i][threadIdx.x];
    grad_bias[col] = s;
}

// ---- the draw -----------------------------------------------------------------------------------------------------------

struct Draw {
    Rows logits;
    int64_t rows, inner;
    int cols;
    const float *uniforms, *temperature, *top_p, *min_p;
    const int32_t *top_k;
    int32_t *tokens;
    float *logprobs;
};

// A float's place in the order of values, as an unsigned number.
__device__ __forceinline__ uint32_t key_of(float z) {
    const uint32_t b = __float_as_uint(z);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

// A value and its column as one number, larger for an earlier rank (a larger value, then a smaller column). 0: none.
__device__ __forceinline__ uint64_t pair_of(float z, int col) { return (uint64_t)key_of(z) << 32 | (uint32_t)~col; }
__device__ __forceinline__ float value_of(uint64_t pair) { return of_key((uint32_t)(pair >> 32)); }
__device__ __forceinline__ int col_of(uint64_t pair) { return (int)~(uint32_t)pair; }

// One workgroup draws from one row, which it reads as often as the filters need (the first time from memory, then from the
// caches: 1000 rows of 65535 floats in 127 us, 2.1 TB/s; kept in registers instead, a row leaves no room for a second
// workgroup on the CU, and 2.3 ms). The usual filters leave few tokens, and those are found without looking at every value
// twice: with NT threads over interleaved columns, the k-th largest of the threads' maxima is no larger than the k-th largest
// value, and little more than k values reach it. They go to one thread each, are sorted, cut, and drawn from. Only where more
// than NT values would have to be looked at (a large k, a flat distribution) the cut is found by histograms over the row.
// What bounds it: the exponentials of rows without top_k (vector instructions issue in 70 % of busy cycles; 44 a value, rows
// with filters counted in). A single row is bound by the latency of one workgroup's steps: 32000 floats, all filters, in 23 us.
template <class T, int NT>
struct Drawer {
    static constexpr int N = Pack<T>::N, W = NT / 64, AHEAD = 4, BINS = 1024;
    struct Shared {
        uint64_t bins[BINS];   // the histogram
        uint64_t list[NT];     // gathered pairs
        uint64_t sorted[NT];   // the same in order
        uint32_t rank[NT];
        double power[256];     // 2^(i / 256)
        uint64_t part[W], low[W], high[W];
        float maxima[W], minima[W];
        int counts[2][W];
        int count, bin, col;
        uint64_t above, cut;
    };
    Shared &sh;
    const T *row;
    int cols;
    float top;      // the row's maximum
    float floor;    // values below it count for nothing
    double scale;   // 256 log2(e) / temperature
    uint64_t cut;   // kept: this pair and larger ones
    bool ones;      // every kept value counts as 1
    double least;   // of the kept values' weights

    // A 64-bit constant in scalar registers, set where it is used: kept through a loop, these constants would push its own
    // values out of the vector registers.
    template <uint64_t BITS>
    __device__ __forceinline__ static double constant() {
        uint32_t low, high;
        asm volatile("s_mov_b32 %0, %1" : "=s"(low) : "i"((uint32_t)BITS));
        asm volatile("s_mov_b32 %0, %1" : "=s"(high) : "i"((uint32_t)(BITS >> 32)));
        return __longlong_as_double((int64_t)((uint64_t)high << 32 | low));
    }
    // ln of the weight in 1 / 256 of a doubling (not above 0: +inf is taken as the largest finite value)
    __device__ __forceinline__ double place_of(float v) const {
        return ((double)fminf(v, 0x1.fffffep127f) - (double)fminf(top, 0x1.fffffep127f)) * scale;
    }
    // exp((v - top) / temperature) = 2^(y / 256), y = n + f with |f| <= 1/2: a power of two, an entry of the table, and four
    // terms of the series of 2^(f / 256), which end below 2^-54. For v >= floor: the power of two is added to the exponent.
    __device__ __forceinline__ double weight(float v) const {
        const double y = place_of(v), magic = constant<0x4338000000000000>();  // 1.5 * 2^52
        const double shifted = y + magic;
        const int n = (int)(uint32_t)__double_as_longlong(shifted);
        const double f = y - (shifted - magic);
        double q = fma(f, constant<0x3d83b2ab6fba4e77>(), constant<0x3e2c6b08d704a0c0>());  // (ln 2 / 256)^n / n!, n = 4, 3
        q = fma(f, q, constant<0x3ecebfbdff82c58f>());                                      // 2
        q = fma(f, q, constant<0x3f662e42fefa39ef>()) * f;                                  // 1
        const double power = __longlong_as_double(__double_as_longlong(sh.power[n & 255]) + ((int64_t)(n >> 8) << 52));
        return fma(power, q, power);
    }
    // 2^47 w rounded: w + 32 has steps of 2^-47, and its mantissa is the multiple
    __device__ __forceinline__ static uint64_t steps(double w) {
        return (uint64_t)__double_as_longlong(w + constant<0x4040000000000000>()) & ((1ull << 52) - 1);
    }
    __device__ __forceinline__ uint64_t mass(float v) const {
        const uint64_t x = steps(weight(v));
        return v >= floor ? x : 0;
    }
    __device__ __forceinline__ uint64_t share(float v, int col) const {
        if (!(v >= floor)) return 0;
        if (cut && pair_of(v, col) < cut) return 0;
        if (ones) return 1;
        const double w = weight(v);
        return w >= least ? steps(w) : 0;
    }
    // What is below the floor weighs nothing (under 2^-48): 36 temperatures down. (Rounding the floor moves it past no value.)
    __device__ __forceinline__ float floor_of(float temperature) const {
        return uniform(top == INF ? INF : fmaxf(top - 36.0f * temperature, -0x1.fffffep127f));
    }
    // NaN counts as -inf; one key for both zeros
    __device__ __forceinline__ static float clean(float z) { return (z == z ? z : -INF) + 0.0f; }

    // f(value, column) over columns from + (t + i * step) * N .. + N, up to `to`; AHEAD packs are on their way at a time
    template <int AHEAD, class F>
    __device__ __forceinline__ void each(int t, int step, int from, int to, F f) {
        int col = from + t * N;
#pragma unroll 1
        for (; col + ((AHEAD - 1) * step + 1) * N <= to; col += AHEAD * step * N) {
            Pack<T> z[AHEAD];
#pragma unroll
            for (int a = 0; a < AHEAD; a++) z[a] = load_pack(row + col + a * step * N);
#pragma unroll
            for (int a = 0; a < AHEAD; a++)
#pragma unroll
                for (int e = 0; e < N; e++) f(clean((float)z[a].v[e]), col + a * step * N + e);
        }
#pragma unroll 1
        for (; col < to; col += step * N) {
            float z[N];
            load_floats<T, N>(row, col, to, -INF, z);
#pragma unroll
            for (int e = 0; e < N; e++)
                if (col + e < to) f(clean(z[e]), col + e);
        }
    }
    template <class F>
    __device__ __forceinline__ void each(F f) {  // the whole row, neighbouring packs by neighbouring threads
        each<4>(threadIdx.x, NT, 0, cols, f);
    }

    // The sum of x over the threads in front of this one; over all in `total`.
    __device__ __forceinline__ uint64_t scan(uint64_t x, uint64_t &total) {
        const int wave = threadIdx.x >> 6;
        const uint64_t in = wave_scan(x);
        __syncthreads();
        if ((threadIdx.x & 63) == 63) sh.part[wave] = in;
        __syncthreads();
        uint64_t at = in - x, all = 0;
#pragma unroll 4
        for (int w = 0; w < W; w++) {
            if (w < wave) at += sh.part[w];
            all += sh.part[w];
        }
        total = all;
        return at;
    }

    // The n pairs of the threads (all different; 0: none), in order, larger first. Each is compared with all others, by NT / n
    // threads: for the few pairs that are sorted here quicker than a network's many steps (1024 pairs: 20 us, 256: 2).
    __device__ __forceinline__ uint64_t sort(uint64_t x, int n) {
        const int t = threadIdx.x;
        int width = 64;
        while (width < n) width <<= 1;
        const int parts = NT / width, each = (n + parts - 1) / parts;
        __syncthreads();
        sh.list[t] = x;
        sh.rank[t] = 0;
        sh.sorted[t] = 0;
        __syncthreads();
        const uint64_t mine = sh.list[t & (width - 1)];
        const int from = t / width * each, to = from + each < n ? from + each : n;
        uint32_t larger = 0;
        int i = from;
        for (; i + 4 <= to; i += 4)
#pragma unroll
            for (int e = 0; e < 4; e++) larger += sh.list[i + e] > mine;
        for (; i < to; i++) larger += sh.list[i] > mine;
        if (larger) atomicAdd(&sh.rank[t & (width - 1)], larger);
        __syncthreads();
        if (x) sh.sorted[sh.rank[t]] = x;
        __syncthreads();
        return sh.sorted[t];
    }
    // How many threads say so. Calls alternate between two places, so that one barrier a call is enough.
    __device__ __forceinline__ int count(bool x, int turn) {
        const int n = __popcll(__ballot(x));
        if ((threadIdx.x & 63) == 0) sh.counts[turn & 1][threadIdx.x >> 6] = n;
        __syncthreads();
        int all = 0;
#pragma unroll 4
        for (int w = 0; w < W; w++) all += sh.counts[turn & 1][w];
        return (int)uniform((uint32_t)all);
    }

    // Waves take the row in contiguous parts: their sums of the shares give the part that t falls into, and the pieces of that
    // part, one for each wave, the place.
    __device__ __forceinline__ int part_size() const { return (cols + W * 64 * N - 1) / (W * 64 * N) * (64 * N); }
    __device__ __forceinline__ uint64_t part_sums() {
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, size = part_size(), from = wave * size;
        uint64_t s = 0, all = 0;
        const int to = from + size < cols ? from + size : cols;
        if (!cut && !ones && least == 0.0) each<1>(lane, 64, from, to, [&](float v, int) { s += mass(v); });
        else each<1>(lane, 64, from, to, [&](float v, int col) { s += share(v, col); });
        s = wave_sum(s);
        __syncthreads();
        if (lane == 0) sh.part[wave] = s;
        __syncthreads();
#pragma unroll 4
        for (int w = 0; w < W; w++) all += sh.part[w];
        return all;
    }
    // After part_sums: leaves in sh.col the first column at which the sum of shares, that column included, exceeds t (t < the total).
    __device__ __forceinline__ void locate(uint64_t t) {
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, size = part_size();
        uint64_t base = 0;
        int part = 0;
        while (t >= base + sh.part[part]) base += sh.part[part++];
        const int from = part * size, to = from + size < cols ? from + size : cols;
        // pieces of 64 * N columns, W at a time
        for (int first = from; first < to; first += W * 64 * N) {
            const int col = first + (wave * 64 + lane) * N;
            uint64_t each[N], s = 0;
            float z[N];
            load_floats<T, N>(row, col, to, -INF, z);
#pragma unroll
            for (int e = 0; e < N; e++) s += each[e] = share(clean(z[e]), col + e);
            uint64_t all, at = base + scan(s, all);
            if (at <= t && t < at + s) {
                bool open = true;
#pragma unroll
                for (int e = 0; e < N; e++) {
                    at += each[e];
                    if (open && at > t) {
                        open = false;
                        sh.col = col + e;
                    }
                }
            }
            base += all;
            if (t < base) break;
        }
        __syncthreads();
    }

    // The pairs that `want` takes, one a thread in any order (0 past them); returns how many there are, which may be more
    // than NT. `mine`: whether this thread's columns can hold any.
    template <class F>
    __device__ __forceinline__ int gather(bool mine, uint64_t &pair, F want) {
        __syncthreads();
        if (threadIdx.x == 0) sh.count = 0;
        __syncthreads();
        auto keep = [&](float v, int col) {
            if (!want(v, col)) return;
            const int i = atomicAdd(&sh.count, 1);
            if (i < NT) sh.list[i] = pair_of(v, col);
        };
        if (mine) each<1>(threadIdx.x, NT, 0, cols, keep);
        __syncthreads();
        const int n = (int)uniform((uint32_t)sh.count);
        pair = (int)threadIdx.x < n ? sh.list[threadIdx.x] : 0;
        return n;
    }

    // Apart from the kernel, whose loops would pay for its registers.
    __device__ __attribute__((noinline)) static uint64_t cut_apart(Shared &sh, const T *row, int cols, float top, float floor, double scale,
                                                                   uint64_t cut, bool ones, uint64_t target, float temperature) {
        Drawer d{sh, row, cols, uniform(top), uniform(floor), uniform(scale), uniform(cut), ones, 0.0};
        d.cut_at(uniform(target), uniform(temperature));
        return d.cut;
    }
    // Moves the cut to the last of the first ranks whose shares sum to `target` or more (0 < target <= the whole sum).
    __device__ __forceinline__ void cut_at(uint64_t target, float temperature) {
        // bins of equal width in value, down to where weights vanish; then within a bin, of equal numbers of pairs
        const float width_inverse = (BINS - 1) / (40.0f * temperature);
        uint64_t low = 0, high = ~0ull, above = 0;
        int shift = -1;  // -1: by value
        for (;;) {
            auto bin_of = [&](float v, uint64_t pair) {
                if (shift < 0) return v == top ? 0 : (int)fminf((top - v) * width_inverse, (float)(BINS - 1));
                return (int)((high - pair) >> shift);
            };
            auto within = [&](float v, uint64_t pair) { return v > -INF && pair >= cut && pair >= low && pair <= high; };
            __syncthreads();
            for (int i = threadIdx.x; i < BINS; i += NT) sh.bins[i] = 0;
            __syncthreads();
            each([&](float v, int col) {
                const uint64_t pair = pair_of(v, col);
                if (within(v, pair)) atomicAdd((unsigned long long *)&sh.bins[bin_of(v, pair)], (unsigned long long)share(v, col));
            });
            __syncthreads();
            constexpr int EACH = BINS / NT;
            uint64_t own[EACH], s = 0, all;
#pragma unroll
            for (int i = 0; i < EACH; i++) s += own[i] = sh.bins[threadIdx.x * EACH + i];
            uint64_t at = above + scan(s, all);
            if (at < target && target <= at + s) {
                bool open = true;
#pragma unroll
                for (int i = 0; i < EACH; i++) {
                    if (open && target <= at + own[i]) {
                        open = false;
                        sh.bin = threadIdx.x * EACH + i;
                        sh.above = at;
                    }
                    at += own[i];
                }
            }
            __syncthreads();
            const int bin = sh.bin;
            above = sh.above;
            // what is in that bin
            uint64_t least_pair = ~0ull, most_pair = 0, pair;
            const int n = gather(true, pair, [&](float v, int col) {
                const uint64_t x = pair_of(v, col);
                const bool in = within(v, x) && bin_of(v, x) == bin;
                if (in) {
                    least_pair = x < least_pair ? x : least_pair;
                    most_pair = x > most_pair ? x : most_pair;
                }
                return in;
            });
            if (n <= NT) {
                pair = sort(pair, n);
                const uint64_t w = pair ? share(value_of(pair), col_of(pair)) : 0;
                const uint64_t from = above + scan(w, all);
                if (from < target && target <= from + w) sh.cut = pair;
                __syncthreads();
                cut = uniform(sh.cut);
                return;
            }
            for (int d = 32; d; d >>= 1) {
                const uint64_t x = __shfl_xor((unsigned long long)least_pair, d), y = __shfl_xor((unsigned long long)most_pair, d);
                least_pair = x < least_pair ? x : least_pair;
                most_pair = y > most_pair ? y : most_pair;
            }
            if ((threadIdx.x & 63) == 0) {
                sh.low[threadIdx.x >> 6] = least_pair;
                sh.high[threadIdx.x >> 6] = most_pair;
            }
            __syncthreads();
            low = ~0ull;
            high = 0;
            for (int w = 0; w < W; w++) {
                low = sh.low[w] < low ? sh.low[w] : low;
                high = sh.high[w] > high ? sh.high[w] : high;
            }
            shift = 0;
            while ((high - low) >> shift >= (uint64_t)BINS) shift++;
        }
    }

    // Draws from the few pairs that can be left by the first k ranks (k > 0), or by the first that sum to `target`; false when
    // that would be more than NT, or not enough.
    __device__ __forceinline__ bool few(float mine, int k, float p, double least_kept, uint64_t target, float u, uint64_t &whole) {
        // a threshold that `wanted` to 1.2 times as many threads' maxima reach
        const int wanted = k > 0 ? k : NT / 4;
        const uint32_t key = key_of(mine);
        float least_mine = sh.minima[0];
#pragma unroll 4
        for (int w = 1; w < W; w++) least_mine = fminf(least_mine, sh.minima[w]);
        uint32_t low = uniform(max(key_of(least_mine), key_of(-INF) + 1)), high = key_of(top);
        for (int i = 0; i < 32 && low < high; i++) {
            const uint32_t mid = low + (high - low) / 2 + 1;
            const int n = count(key >= mid, i);
            if (n < wanted) high = mid - 1;
            else {
                low = mid;
                if (n <= wanted + wanted / 5) break;
            }
        }
        uint64_t pair, all;
        const int n = gather(key >= low, pair, [&](float v, int) { return key_of(v) >= low; });
        if (n > NT) return false;
        pair = sort(pair, n);
        const bool in = pair && (k <= 0 || (int)threadIdx.x < k);
        const bool weighs = in && value_of(pair) >= floor;
        const double w = weighs ? weight(value_of(pair)) : 0.0;
        const uint64_t at = scan(weighs ? steps(w) : 0, all);
        if (k > 0) target = target_of(p, all);
        else if (all < target) return false;
        const bool keep = in && (p >= 1.0f || at < target) && w >= least_kept;
        const int left = count(keep, 0);  // (they are the first ones)
        const uint64_t by_id = sort(keep ? pair << 32 | pair >> 32 : 0, left);
        const float v = of_key((uint32_t)by_id);
        const uint64_t s = by_id ? mass(v) : 0;
        const uint64_t from = scan(s, whole), t = part_of_whole(u, whole);
        if (from <= t && t < from + s) sh.col = (int)~(uint32_t)(by_id >> 32);
        __syncthreads();
        return true;
    }
    __device__ __forceinline__ static uint64_t target_of(float p, uint64_t whole) {
        const uint64_t t = (uint64_t)ceil((double)p * (double)whole);
        return t < 1 ? 1 : t > whole ? whole : t;
    }

    // floor(u * whole) without rounding (below the whole): u = m * 2^-n with 24 bits of m, which stand at the product's top
    __device__ __forceinline__ static uint64_t part_of_whole(float u, uint64_t whole) {
        if (u >= 1.0f) return whole - 1;
        if (!(u >= 0x1p-126f)) return 0;  // (the whole is below 2^64)
        const uint32_t b = __float_as_uint(u), n = 126 - (b >> 23);  // u = 1/2 .. 1 times 2^-n
        return __umul64hi(whole, (uint64_t)(b << 8 | 0x80000000u) << 32) >> min(n, 63u);
    }

    __device__ __forceinline__ void draw(const Draw &a, int64_t r) {
        const float temperature = a.temperature ? a.temperature[r] : 1.0f, p = a.top_p ? a.top_p[r] : 1.0f;
        const float least_f = a.min_p ? a.min_p[r] : 0.0f, u = uniform(a.uniforms[r]);
        const int k = a.top_k ? a.top_k[r] : 0;
        // the maximum of this thread's columns, and the first column that holds it
        float mine = -INF;
        int place = 0;
        each([&](float v, int col) {
            if (v > mine) {
                mine = v;
                place = col;
            }
        });
        top = wave_max(mine);
        const float lowest = -wave_max(-mine);
        if ((threadIdx.x & 63) == 0) {
            sh.maxima[threadIdx.x >> 6] = top;
            sh.minima[threadIdx.x >> 6] = lowest;
        }
        if (threadIdx.x == 0) sh.col = cols;
        __syncthreads();
#pragma unroll 4
        for (int w = 0; w < W; w++) top = fmaxf(top, sh.maxima[w]);
        top = uniform(top);
        if (!(top > -INF)) {
            if (threadIdx.x == 0) {
                a.tokens[r] = -1;
                if (a.logprobs) a.logprobs[r] = -INF;
            }
            return;
        }
        if (!(temperature > 0.0f) || k == 1 || p <= 0.0f) {  // the first rank
            if (mine == top) atomicMin(&sh.col, place);
            __syncthreads();
            if (threadIdx.x == 0) {
                a.tokens[r] = sh.col;
                if (a.logprobs) a.logprobs[r] = 0.0f;
            }
            return;
        }
        scale = uniform(256 * 0x1.71547652b82fep0 / (double)temperature);
        cut = 0;
        const double least_kept = uniform(least_f > 0.0f ? least_f < 1.0f ? (double)least_f : 1.0 : 0.0);
        const bool by_k = k > 0 && k < cols, by_p = p < 1.0f;
        bool untried = !by_k || k <= NT * 5 / 8;
        uint64_t whole;
        // 0: the cut by rank, 1: by share, 2: the draw from what is left
        for (int stage = by_k ? 0 : by_p ? 1 : 2;;) {
            ones = stage == 0;
            floor = ones ? -0x1.fffffep127f : floor_of(temperature);
            least = stage == 2 ? least_kept : 0.0;
            const bool sums = stage || !untried;
            if (sums) whole = uniform(part_sums());
            if (stage == 2) {
                locate(part_of_whole(u, whole));
                break;
            }
            const uint64_t target = stage ? target_of(p, whole) : (uint64_t)k;
            if (untried) {
                untried = false;
                uint64_t left;
                floor = floor_of(temperature);
                if (few(mine, by_k ? k : 0, p, least_kept, target, u, left)) {
                    whole = left;
                    break;
                }
                if (!sums) continue;
            }
            if (target < whole) cut = uniform(cut_apart(sh, row, cols, top, floor, scale, cut, ones, target, temperature));
            stage = stage == 0 && by_p ? 1 : 2;
        }
        if (threadIdx.x == 0) {
            const int col = sh.col;
            a.tokens[r] = col;
            if (a.logprobs) {
                const double x = place_of(clean((float)row[col])) * (0x1.62e42fefa39efp-1 / 256);
                a.logprobs[r] = (float)(x - log((double)whole * 0x1p-47));
            }
        }
    }
};

template <class T, int NT, int WAVES>
__global__ __launch_bounds__(NT, WAVES) void draw_kernel(Draw a, int64_t first) {
    using D = Drawer<T, NT>;
    __shared__ typename D::Shared sh;
    if (threadIdx.x < 256) sh.power[threadIdx.x] = exp2((double)threadIdx.x / 256);
    const int64_t r = first + blockIdx.x;
    D{sh, row_of<T>(a.logits, r, a.inner), a.cols, 0.0f, 0.0f, 0.0, 0, false, 0.0}.draw(a, r);
}

// ---- log-probabilities --------------------------------------------------------------------------------------------------

struct Logprobs {
    Rows logits, grad_logits;
    int64_t rows, inner;
    int cols, wide_ids;
    const void *tokens;
    const float *temperature, *grad;
    float *logprobs, *stats;
};

constexpr float LOG2E = 1.44269504088896340736f;

__device__ __forceinline__ int64_t token_of(const Logprobs &a, int64_t r) {
    return a.wide_ids ? ((const int64_t *)a.tokens)[r] : (int64_t)((const int32_t *)a.tokens)[r];
}

// 1 / temperature. What is below 2^-126, or not positive at all, counts as 2^-126; for an infinite one the least float stands
// in place of 0, whose product with -inf would be NaN (any finite exponent is then below 2^-20).
__device__ __forceinline__ float inverse_of(float temperature) { return fmaxf(1.0f / fmaxf(temperature, 0x1p-126f), 0x1p-149f); }
// Half of z - top: the difference itself may be past what 32 bits hold (3e38 - -3e38) where temperatures are high. The same
// bits as z - top otherwise.
__device__ __forceinline__ float half_below(float z, float half_top) { return fmaf(z, 0.5f, -half_top); }

// exp((z - top) / temperature) = 2^(d * scale), d half of z - top. The sum of a row takes the product rounded once: that is off by
// a few 2^-24 of the mean of -d * scale under the softmax, which is below log2 of the columns. An element of the gradient would be
// off by 2^-24 for each doubling that its own z lies below the top; where it is written in 32 bits the product is taken in two
// parts, d * (scale + low). (In the sum too: 19 us become 21 for 20000 rows of 1000 floats.)
struct Exponent {
    float scale, low;
    __device__ __forceinline__ Exponent(float temperature, float inverse) : scale(2 * (inverse * LOG2E)) {
        // 1 / temperature = inverse + inverse * more; 2 * LOG2E + what its 24 bits leave out
        const float t = fmaxf(temperature, 0x1p-126f), more = t < 0x1p126f ? fmaf(-t, inverse, 1.0f) : 0.0f;
        low = fmaf(2 * LOG2E, inverse, -scale) + fmaf(scale, more, inverse * 3.851925982e-8f);
    }
    __device__ __forceinline__ float power(float d) const { return __builtin_amdgcn_exp2f(d * scale); }
    __device__ __forceinline__ float exact_power(float d) const {
        const float x = d * scale, y = __builtin_amdgcn_exp2f(x);
        const float rest = fmaf(d, low, fmaf(d, scale, -x));  // NaN where x is infinite: y is 0 there
        return fmaf(y, fminf(fmaxf(rest, -1.0f), 1.0f) * 0.693147181f, y);
    }
};

// One pass with a running maximum and sum. TPR threads go over one row, AHEAD loads of 16 bytes each at a time. 8192 rows of 32000
// bf16 in 121 us (0.52 GB, 4.3 TB/s; with one load at a time the kernel took 1.37 times as long). Short rows take a wave each. Bound
// by memory.
template <class T, int TPR>
__global__ __launch_bounds__(256) void logprobs_kernel(Logprobs a) {
    constexpr int N = Pack<T>::N, PER = 256 / TPR, AHEAD = 4;
    __shared__ float maxima[4], sums[4];
    const int t = threadIdx.x % TPR;
    for (int64_t r0 = blockIdx.x * (int64_t)PER; r0 < a.rows; r0 += gridDim.x * (int64_t)PER) {
        const int64_t r = r0 + threadIdx.x / TPR;
        const bool on = r < a.rows;
        const float temperature = on && a.temperature ? a.temperature[r] : 1.0f;
        const float inverse = inverse_of(temperature);
        const Exponent exponent(temperature, inverse);
        const T *row = on ? row_of<T>(a.logits, r, a.inner) : nullptr;
        float m = -INF, s = 0.0f;
        auto add = [&](const float *z, int n) {
            float more = m;
#pragma unroll
            for (int e = 0; e < n; e++) more = fmaxf(more, z[e]);
            const float from = more == -INF ? 0.0f : 0.5f * more;  // (nothing yet above -inf: the exponentials are 0, not NaN)
            s *= exponent.power(half_below(m, from));
#pragma unroll
            for (int e = 0; e < n; e++) s += exponent.power(half_below(z[e], from));
            m = more;
        };
        if (on) {
            int col = t * N;
#pragma unroll 1
            for (; col + ((AHEAD - 1) * TPR + 1) * N <= a.cols; col += AHEAD * TPR * N) {
                Pack<T> x[AHEAD];
#pragma unroll
                for (int i = 0; i < AHEAD; i++) x[i] = load_pack(row + col + i * TPR * N);
                float z[AHEAD * N];
#pragma unroll
                for (int i = 0; i < AHEAD * N; i++) z[i] = (float)x[i / N].v[i % N];
                add(z, AHEAD * N);
            }
#pragma unroll 1
            for (; col < a.cols; col += TPR * N) {
                float z[N];
                load_floats<T, N>(row, col, a.cols, -INF, z);
                add(z, N);
            }
        }
        float top = wave_max(m);
        s = wave_sum(s * exponent.power(half_below(m, top == -INF ? 0.0f : 0.5f * top)));
        if (TPR > 64) {
            __syncthreads();
            if ((threadIdx.x & 63) == 0) {
                maxima[threadIdx.x >> 6] = top;
                sums[threadIdx.x >> 6] = s;
            }
            __syncthreads();
            top = fmaxf(fmaxf(maxima[0], maxima[1]), fmaxf(maxima[2], maxima[3]));
            const float from = top == -INF ? 0.0f : 0.5f * top;
            s = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; w++) s += sums[w] * exponent.power(half_below(maxima[w], from));
        }
        if (on && t == 0) {
            const int64_t token = token_of(a, r);
            float y = 0.0f;
            if (token >= a.cols) y = __builtin_nanf("");
            else if (token >= 0) y = s == 0.0f ? -INF : half_below((float)row[token], 0.5f * top) * (2 * inverse) - logf(s);
            a.logprobs[r] = y;
            if (a.stats) {
                a.stats[2 * r] = top;
                a.stats[2 * r + 1] = s;
            }
        }
    }
}

// One slice of columns (blockIdx.y) of one row after another. 8192 rows of 32000 bf16 in 189 us (1.05 GB read and written, 5.5 TB/s
// with what the caches keep of the forward pass; the loads come before the scalars that they do not need). Bound by memory.
template <class T>
__global__ __launch_bounds__(256) void logprobs_grad_kernel(Logprobs a) {
    constexpr int N = Pack<T>::N, C = 2;
    const int first = blockIdx.y * 256 * C * N + threadIdx.x * N;
    for (int64_t i = blockIdx.x; i < a.rows; i += gridDim.x) {
        const int64_t r = a.rows - 1 - i;  // what the forward pass read last may still be in the cache
        const T *row = row_of<T>(a.logits, r, a.inner);
        T *out = row_of<T>(a.grad_logits, r, a.inner);
        Raw<T, N> x[C];
#pragma unroll
        for (int c = 0; c < C; c++) x[c].load(row, first + c * 256 * N, a.cols);
        const int64_t token = token_of(a, r);
        const float temperature = a.temperature ? a.temperature[r] : 1.0f;
        const float inverse = inverse_of(temperature);
        const Exponent exponent(temperature, inverse);
        const float half_top = 0.5f * a.stats[2 * r], s = a.stats[2 * r + 1];
        const bool scored = token >= 0 && s != 0.0f;
        const float g = scored ? a.grad[r] * inverse : 0.0f;
        const float less = token >= a.cols ? __builtin_nanf("") : g / s;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int col = first + c * 256 * N;
            if (col >= a.cols) continue;
            float z[N];
#pragma unroll
            for (int e = 0; e < N; e++) {
                const float below = half_below(x[c].get(e), half_top);
                const float d = scored ? -less * (sizeof(T) == 4 ? exponent.exact_power(below) : exponent.power(below)) : 0.0f;
                z[e] = col + e == token ? g + d : d;
            }
            store_floats<T, N>(out, col, a.cols, z);
        }
    }
}

// ---- launches -----------------------------------------------------------------------------------------------------------

// The caller's device for the launch, and what was current before it.
struct OnDevice {
    int was = -1;
    bool moved = false;
    zbpe_status go(int device) {
        if (hipGetDevice(&was) != hipSuccess) return refuse(ZBPE_DEVICE_ERROR, "no HIP device");
        if (was == device) return ZBPE_OK;
        const hipError_t e = hipSetDevice(device);
        if (e != hipSuccess) return refuse(ZBPE_DEVICE_ERROR, "device %d: %s", device, hipGetErrorString(e));
        moved = true;
        return ZBPE_OK;
    }
    ~OnDevice() {
        if (moved) (void)hipSetDevice(was);
    }
};

static zbpe_status launched(const char *what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? ZBPE_OK : refuse(ZBPE_DEVICE_ERROR, "%s: %s", what, hipGetErrorString(e));
}

// Workgroups of a launch over `items`: each goes on by the grid's size, so any number of items is covered.
static unsigned grid_of(int64_t items) { return (unsigned)(items < (1 << 21) ? items : (1 << 21)); }

static bool is_float(int dtype) { return dtype == ZBPE_F32 || dtype == ZBPE_F16 || dtype == ZBPE_BF16; }
static Rows rows_of(const zbpe_rows &m) { return Rows{(char *)m.data, m.outer_stride, m.inner_stride}; }

static zbpe_status check_rows(const char *what, int64_t rows, int64_t inner, int cols) {
    if (cols < 1 || cols > ZBPE_MAX_VOCAB) return refuse(ZBPE_INVALID_ARGUMENT, "%s: %d columns (1 to %d)", what, cols, ZBPE_MAX_VOCAB);
    if (rows < 0 || rows >= (1ll << 40)) return refuse(ZBPE_INVALID_ARGUMENT, "%s: %lld rows", what, (long long)rows);
    if (inner < 1) return refuse(ZBPE_INVALID_ARGUMENT, "%s: inner is %lld", what, (long long)inner);
    return ZBPE_OK;
}
static zbpe_status check_matrix(const char *what, const char *name, const zbpe_rows &m, int64_t rows) {
    if (!is_float(m.dtype)) return refuse(ZBPE_INVALID_ARGUMENT, "%s: %s has data type %d (F32, F16 or BF16)", what, name, m.dtype);
    if (!m.data && rows) return refuse(ZBPE_INVALID_ARGUMENT, "%s: no %s", what, name);
    return ZBPE_OK;
}
// rows that are written: none of them overlaps another
static zbpe_status check_written(const char *what, const char *name, const zbpe_rows &m, int64_t rows, int64_t inner, int cols) {
    const zbpe_status s = check_matrix(what, name, m, rows);
    if (s != ZBPE_OK) return s;
    const int64_t n_inner = rows < inner ? rows : inner, n_outer = rows / inner + (rows % inner != 0);
    int64_t a = m.inner_stride < 0 ? -m.inner_stride : m.inner_stride, b = m.outer_stride < 0 ? -m.outer_stride : m.outer_stride;
    const bool ok = (n_inner < 2 || a >= cols) && (n_outer < 2 || b >= cols) &&
                    (n_inner < 2 || n_outer < 2 || b >= a * (n_inner - 1) + cols || a >= b * (n_outer - 1) + cols);
    return ok ? ZBPE_OK : refuse(ZBPE_INVALID_ARGUMENT, "%s: the rows of %s overlap", what, name);
}

// The memory of a matrix or an array: n[0] * n[1] pieces of `size` bytes, step[0] and step[1] bytes apart, step[0] >= step[1].
using wide = __int128;
struct Pieces {
    wide from = 0, size = 0, step[2] = {1, 1}, n[2] = {0, 0};  // no pieces

    static Pieces array(const void *data, wide bytes) {
        Pieces p;
        if (!data || bytes <= 0) return p;
        p.from = (wide)(uintptr_t)data;
        p.size = bytes;
        p.n[0] = p.n[1] = 1;
        return p;
    }
    static Pieces rows(const void *data, wide bytes, int64_t n_outer, wide outer_step, int64_t n_inner, wide inner_step) {
        Pieces p = array(data, bytes);
        if (!p.size || n_outer < 1 || n_inner < 1) return Pieces();
        const int64_t n[2] = {n_outer, n_inner};
        const wide steps[2] = {outer_step, inner_step};
        for (int i = 0; i < 2; i++) {
            p.n[i] = n[i];
            p.step[i] = steps[i];
            if (p.step[i] < 0) p.from += p.step[i] * (p.n[i] - 1);
            if (p.step[i] < 0) p.step[i] = -p.step[i];
            if (p.step[i] == 0 || p.n[i] == 1) p.n[i] = p.step[i] = 1;
        }
        if (p.step[0] < p.step[1]) {
            std::swap(p.step[0], p.step[1]);
            std::swap(p.n[0], p.n[1]);
        }
        return p;
    }
    wide end() const { return from + step[0] * (n[0] - 1) + step[1] * (n[1] - 1) + size; }
    bool operator==(const Pieces &o) const {
        return from == o.from && size == o.size && n[0] == o.n[0] && n[1] == o.n[1] && (n[0] == 1 || step[0] == o.step[0]) && (n[1] == 1 || step[1] == o.step[1]);
    }
    // Whether one of these pieces starts within lo .. hi. Few i need a look where the pieces of one i end before the next i's.
    bool starts_within(wide lo, wide hi) const {
        lo -= from;
        hi -= from;
        const wide before = lo - step[1] * (n[1] - 1);
        for (wide i = before > 0 ? (before + step[0] - 1) / step[0] : 0; i < n[0] && i * step[0] <= hi; i++) {
            const wide at = lo - i * step[0];
            const wide j = at > 0 ? (at + step[1] - 1) / step[1] : 0;
            if (j < n[1] && i * step[0] + j * step[1] <= hi) return true;
        }
        return false;
    }
    // Whether any byte is in both; these pieces are apart from each other (check_written).
    bool meets(const Pieces &o) const {
        if (!n[0] || !o.n[0] || end() <= o.from || o.end() <= from) return false;
        if (step[0] == o.step[0] && step[1] == o.step[1] && n[0] == o.n[0] && n[1] == o.n[1]) {
            // rows of one kind: by the distances between two of them
            Pieces d = *this;
            for (int i = 0; i < 2; i++) {
                d.from -= d.step[i] * (d.n[i] - 1);
                d.n[i] = 2 * d.n[i] - 1;
            }
            return d.starts_within(o.from - size + 1, o.from + o.size - 1);
        }
        for (wide i = 0; i < o.n[0]; i++)
            for (wide j = 0; j < o.n[1]; j++) {
                const wide at = o.from + i * o.step[0] + j * o.step[1];
                if (starts_within(at - size + 1, at + o.size - 1)) return true;
            }
        return false;
    }
};
// A matrix: its whole outer steps, and the rows of one that is not whole.
struct Memory {
    Pieces part[2];
    Memory() = default;
    Memory(const void *data, wide bytes) : part{Pieces::array(data, bytes), Pieces()} {}
    Memory(const zbpe_rows &m, int64_t rows, int64_t inner, int64_t cols) {
        const int element = m.dtype == ZBPE_F32 || m.dtype == ZBPE_I32 ? 4 : m.dtype == ZBPE_I64 ? 8 : 2;
        const wide bytes = (wide)cols * element, outer = (wide)m.outer_stride * element, step = (wide)m.inner_stride * element;
        part[0] = Pieces::rows(m.data, bytes, rows / inner, outer, inner, step);
        part[1] = Pieces::rows(m.data, bytes, 1, 1, rows % inner, step);
        if (part[1].n[0]) part[1].from += outer * (rows / inner);
    }
    bool operator==(const Memory &o) const { return part[0] == o.part[0] && part[1] == o.part[1]; }
    bool meets(const Memory &o) const {
        return part[0].meets(o.part[0]) || part[0].meets(o.part[1]) || part[1].meets(o.part[0]) || part[1].meets(o.part[1]);
    }
};
static zbpe_status apart(const char *what, const char *written, const Memory &w, const char *read, const Memory &r) {
    return w.meets(r) ? refuse(ZBPE_INVALID_ARGUMENT, "%s: %s overlaps %s", what, written, read) : ZBPE_OK;
}

// The memory `w` that a call of adjust_logits or its gradient writes, against what it reads besides the logits.
static zbpe_status apart_from_terms(const char *what, const char *written, const Memory &w, const zbpe_adjust &p) {
    const wide rows = p.rows;
    struct {
        const char *name;
        Memory r;
    } const read[] = {
        {"history", p.history_len ? Memory(p.history, p.rows, p.inner, p.history_len) : Memory()},
        {"lengths", Memory(p.lengths, rows * 4)},
        {"prompt_lengths", Memory(p.prompt_lengths, rows * 4)},
        {"repetition", Memory(p.repetition, rows * 4)},
        {"presence", Memory(p.presence, rows * 4)},
        {"frequency", Memory(p.frequency, rows * 4)},
        {"bias", Memory(p.bias, (wide)p.cols * 4)},
        {"bias_tokens", Memory(p.bias_tokens, rows * p.n_biases * 4)},
        {"bias_values", Memory(p.bias_values, rows * p.n_biases * 4)},
        {"masks", Memory(p.masks, (wide)p.mask_rows * p.mask_words * 4)},
        {"states", Memory(p.masks ? p.states : nullptr, rows * 4)},
    };
    for (const auto &x : read) {
        const zbpe_status s = apart(what, written, w, x.name, x.r);
        if (s != ZBPE_OK) return s;
    }
    return ZBPE_OK;
}

template <class F>
static zbpe_status by_type(int dtype, F f) {
    return dtype == ZBPE_F32 ? f(float()) : dtype == ZBPE_F16 ? f(f16()) : f(bf16());
}

static zbpe_status grammar_of(const char *what, const zbpe_grammar *g, int64_t rows, Automaton *out) {
    if (!g) return refuse(ZBPE_INVALID_ARGUMENT, "%s: no grammar", what);
    if (g->vocab_size < 1 || g->vocab_size > ZBPE_MAX_VOCAB)
        return refuse(ZBPE_INVALID_ARGUMENT, "%s: a vocabulary of %d (1 to %d)", what, g->vocab_size, ZBPE_MAX_VOCAB);
    if (g->end_token < -1 || g->end_token >= g->vocab_size) return refuse(ZBPE_INVALID_ARGUMENT, "%s: end token %d", what, g->end_token);
    if (g->n_states < 0 || g->n_states >= (1 << 23)) return refuse(ZBPE_INVALID_ARGUMENT, "%s: %d states (fewer than 2^23)", what, g->n_states);
    if (rows < 0 || rows >= (1ll << 40)) return refuse(ZBPE_INVALID_ARGUMENT, "%s: %lld rows", what, (long long)rows);
    if (!g->offsets || !g->bytes || (!g->next && g->n_states)) return refuse(ZBPE_INVALID_ARGUMENT, "%s: an array of the grammar is missing", what);
    *out = Automaton{g->offsets, g->bytes, g->next, g->accepting, g->index, g->vocab_size, g->end_token, g->n_states};
    return ZBPE_OK;
}

// Rows of one workgroup: as many workgroups as run at a time share the rows evenly (a second, partly filled turn would cost as
// much as a full one), up to ADJUST_RUN rows each. More rows mean fewer loads of the shared bias, and fewer partial sums of its
// gradient to write and add.
template <class T>
static void adjust_plan(int64_t rows, int cols, Adjust *a) {
    constexpr int64_t groups = 256 * ADJUST_GROUPS;
    a->slices = (cols + ADJUST_SLICE<T> - 1) / ADJUST_SLICE<T>;
    const int64_t fit = (rows * a->slices + groups - 1) / groups;
    a->run = (int)(fit < 1 ? 1 : fit > ADJUST_RUN ? ADJUST_RUN : fit);
    a->runs = (rows + a->run - 1) / a->run;
}

static zbpe_status adjust_of(const char *what, const zbpe_adjust *p, Adjust *out) {
    if (!p) return refuse(ZBPE_INVALID_ARGUMENT, "%s: no arguments", what);
    if (p->struct_size != sizeof(zbpe_adjust)) return refuse(ZBPE_INVALID_ARGUMENT, "%s: arguments of another version", what);
    zbpe_status s = check_rows(what, p->rows, p->inner, p->cols);
    if (s == ZBPE_OK) s = check_matrix(what, "logits", p->logits, p->rows);
    if (s != ZBPE_OK) return s;
    if (p->out.dtype != p->logits.dtype && p->out.dtype != ZBPE_F32)
        return refuse(ZBPE_INVALID_ARGUMENT, "%s: out has the type of the logits, or F32", what);
    if (p->history_len < 0 || (p->history.data && p->history.dtype != ZBPE_I32 && p->history.dtype != ZBPE_I64))
        return refuse(ZBPE_INVALID_ARGUMENT, "%s: a history of %lld tokens of data type %d (I32 or I64)", what, (long long)p->history_len, p->history.dtype);
    if (p->history_len >= (1ll << 31)) return refuse(ZBPE_INVALID_ARGUMENT, "%s: a history of 2^31 tokens or more", what);
    if (p->n_biases < 0 || p->n_biases > ZBPE_MAX_BIASES) return refuse(ZBPE_INVALID_ARGUMENT, "%s: %d biases (0 to %d)", what, p->n_biases, ZBPE_MAX_BIASES);
    if (p->n_biases && p->rows && (!p->bias_tokens || !p->bias_values)) return refuse(ZBPE_INVALID_ARGUMENT, "%s: bias tokens without values, or values without tokens", what);
    if (p->masks) {
        if (p->mask_words < (p->cols + 31) / 32) return refuse(ZBPE_INVALID_ARGUMENT, "%s: %d words of mask for %d columns", what, p->mask_words, p->cols);
        if (p->mask_rows < 0 || (!p->states && p->mask_rows != 1 && p->mask_rows < p->rows))
            return refuse(ZBPE_INVALID_ARGUMENT, "%s: %lld rows of masks for %lld rows", what, (long long)p->mask_rows, (long long)p->rows);
    }
    Adjust a{};
    a.logits = rows_of(p->logits);
    a.out = rows_of(p->out);
    if (p->history_len) a.history = rows_of(p->history);
    a.wide_ids = p->history.dtype == ZBPE_I64;
    a.rows = p->rows;
    a.inner = p->inner;
    a.cols = p->cols;
    a.history_len = p->history_len;
    a.lengths = p->lengths;
    a.prompt_lengths = p->prompt_lengths;
    a.repetition = p->repetition;
    a.presence = p->presence;
    a.frequency = p->frequency;
    a.bias = p->bias;
    a.bias_tokens = p->bias_tokens;
    a.bias_values = p->bias_values;
    a.n_biases = p->n_biases;
    a.masks = p->masks;
    a.words = p->mask_words;
    a.mask_rows = p->mask_rows;
    a.states = p->states;
    *out = a;
    return ZBPE_OK;
}

// One row a workgroup, without a loop over rows in the kernel: what such a loop keeps in registers for the next row costs it
// half its waves.
template <class T>
static void draw_launch(const Draw &a, hipStream_t stream) {
    for (int64_t first = 0; first < a.rows; first += 1 << 21) {
        const unsigned grid = (unsigned)(a.rows - first < (1 << 21) ? a.rows - first : 1 << 21);
        if (a.cols <= 1024) draw_kernel<T, 256, 8><<<grid, 256, 0, stream>>>(a, first);
        else draw_kernel<T, 1024, 8><<<grid, 1024, 0, stream>>>(a, first);
    }
}

static zbpe_status logprobs_of(const char *what, const zbpe_logprobs *p, Logprobs *out) {
    if (!p) return refuse(ZBPE_INVALID_ARGUMENT, "%s: no arguments", what);
    if (p->struct_size != sizeof(zbpe_logprobs)) return refuse(ZBPE_INVALID_ARGUMENT, "%s: arguments of another version", what);
    zbpe_status s = check_rows(what, p->rows, p->inner, p->cols);
    if (s == ZBPE_OK) s = check_matrix(what, "logits", p->logits, p->rows);
    if (s != ZBPE_OK) return s;
    if (p->tokens_dtype != ZBPE_I32 && p->tokens_dtype != ZBPE_I64)
        return refuse(ZBPE_INVALID_ARGUMENT, "%s: tokens of data type %d (I32 or I64)", what, p->tokens_dtype);
    if (!p->tokens && p->rows) return refuse(ZBPE_INVALID_ARGUMENT, "%s: no tokens", what);
    *out = Logprobs{rows_of(p->logits), {}, p->rows, p->inner, p->cols, p->tokens_dtype == ZBPE_I64, p->tokens, p->temperature, nullptr, p->logprobs, p->stats};
    return ZBPE_OK;
}

}  // namespace zbpe

using namespace zbpe;

extern "C" {

size_t zbpe_struct_size(int which) {
    return which == 0 ? sizeof(zbpe_adjust) : which == 1 ? sizeof(zbpe_draw) : which == 2 ? sizeof(zbpe_logprobs) : which == 3 ? sizeof(zbpe_grammar) : 0;
}

zbpe_status zbpe_vocab_bytes(const uint16_t *triples, size_t n_merges, size_t vocab_size, uint32_t *offsets, uint8_t *bytes,
                             size_t cap, size_t *n_bytes) {
    if ((!triples && n_merges) || !offsets || !n_bytes || (!bytes && cap)) return refuse(ZBPE_INVALID_ARGUMENT, "zbpe_vocab_bytes: an array is missing");
    if (vocab_size < 256 || vocab_size > ZBPE_MAX_VOCAB)
        return refuse(ZBPE_INVALID_ARGUMENT, "zbpe_vocab_bytes: a vocabulary of %zu (256 to %d)", vocab_size, ZBPE_MAX_VOCAB);
    try {
        VocabTree tree;
        const zbpe_status s = tree.build(triples, n_merges, vocab_size);
        if (s != ZBPE_OK) return refuse(s, "zbpe_vocab_bytes: %s", tree.err.c_str());
        *n_bytes = (size_t)tree.total;
        tree.write(offsets, cap >= tree.total ? bytes : nullptr);
        return ZBPE_OK;
    } catch (const std::bad_alloc &) {
        return refuse(ZBPE_OUT_OF_MEMORY, "zbpe_vocab_bytes: out of host memory");
    } catch (const std::exception &e) {
        return refuse(ZBPE_INTERNAL, "zbpe_vocab_bytes: %s", e.what());
    }
}

size_t zbpe_vocab_index_size(size_t vocab_size) { return vocab_size < 1 || vocab_size > ZBPE_MAX_VOCAB ? 0 : index_size(vocab_size); }

zbpe_status zbpe_vocab_index(const uint32_t *offsets, const uint8_t *bytes, size_t vocab_size, void *index) {
    if (!offsets || !bytes || !index) return refuse(ZBPE_INVALID_ARGUMENT, "zbpe_vocab_index: an array is missing");
    if (vocab_size < 1 || vocab_size > ZBPE_MAX_VOCAB)
        return refuse(ZBPE_INVALID_ARGUMENT, "zbpe_vocab_index: a vocabulary of %zu (1 to %d)", vocab_size, ZBPE_MAX_VOCAB);
    for (size_t v = 0; v < vocab_size; v++)
        if (offsets[v] > offsets[v + 1]) return refuse(ZBPE_INVALID_ARGUMENT, "zbpe_vocab_index: the offsets of token %zu fall", v);
    try {
        index_tokens(offsets, bytes, vocab_size, index);
        return ZBPE_OK;
    } catch (const std::bad_alloc &) {
        return refuse(ZBPE_OUT_OF_MEMORY, "zbpe_vocab_index: out of host memory");
    }
}

zbpe_status zbpe_grammar_masks(int device, void *stream, const zbpe_grammar *grammar, const int32_t *states, int64_t rows,
                               uint32_t *masks) {
    const char *what = "zbpe_grammar_masks";
    Automaton g;
    zbpe_status s = grammar_of(what, grammar, rows, &g);
    if (s != ZBPE_OK || !rows) return s;
    if (!masks) return refuse(ZBPE_INVALID_ARGUMENT, "%s: no masks", what);
    if (!g.index) return refuse(ZBPE_INVALID_ARGUMENT, "%s: no index of the tokens", what);
    const Memory written(masks, (wide)rows * ((g.vocab + 31) / 32) * 4);
    s = apart(what, "masks", written, "states", Memory(states, (wide)rows * 4));
    if (s == ZBPE_OK) s = apart(what, "masks", written, "the automaton", Memory(g.next, (wide)g.n * 1024));
    if (s == ZBPE_OK) s = apart(what, "masks", written, "the automaton", Memory(g.accepting, g.n));
    if (s == ZBPE_OK) s = apart(what, "masks", written, "the index of the tokens", Memory(g.index, (wide)index_size(g.vocab)));
    if (s != ZBPE_OK) return s;
    OnDevice on;
    if ((s = on.go(device)) != ZBPE_OK) return s;
    // a workgroup's slices share what it finds out about its state; few rows need many workgroups
    const int slices = (g.vocab + INDEX_SLICE - 1) / INDEX_SLICE;
    const int64_t fit = rows * slices / 4096;
    const int per = (int)(fit < 1 ? 1 : fit < slices ? fit : slices);
    const int64_t parts = rows * ((slices + per - 1) / per);
    if (parts < 512) grammar_masks_kernel<1024><<<grid_of(parts), 1024, 0, (hipStream_t)stream>>>(g, states, rows, masks, slices, per);
    else grammar_masks_kernel<512><<<grid_of(parts), 512, 0, (hipStream_t)stream>>>(g, states, rows, masks, slices, per);
    return launched(what);
}

zbpe_status zbpe_grammar_advance(int device, void *stream, const zbpe_grammar *grammar, const int32_t *states,
                                 const int32_t *tokens, int64_t rows, int32_t *out) {
    const char *what = "zbpe_grammar_advance";
    Automaton g;
    zbpe_status s = grammar_of(what, grammar, rows, &g);
    if (s != ZBPE_OK || !rows) return s;
    if (!states || !tokens || !out) return refuse(ZBPE_INVALID_ARGUMENT, "%s: an array is missing", what);
    const Memory written(out, (wide)rows * 4);
    if (out != states) s = apart(what, "out", written, "states", Memory(states, (wide)rows * 4));
    if (s == ZBPE_OK && out != tokens) s = apart(what, "out", written, "tokens", Memory(tokens, (wide)rows * 4));
    if (s == ZBPE_OK) s = apart(what, "out", written, "the automaton", Memory(g.next, (wide)g.n * 1024));
    if (s == ZBPE_OK) s = apart(what, "out", written, "the automaton", Memory(g.accepting, g.n));
    if (s != ZBPE_OK) return s;
    OnDevice on;
    if ((s = on.go(device)) != ZBPE_OK) return s;
    grammar_advance_kernel<<<grid_of((rows + 255) / 256), 256, 0, (hipStream_t)stream>>>(g, states, tokens, rows, out);
    return launched(what);
}

zbpe_status zbpe_adjust_logits(int device, void *stream, const zbpe_adjust *args) {
    const char *what = "zbpe_adjust_logits";
    Adjust a;
    zbpe_status s = adjust_of(what, args, &a);
    if (s == ZBPE_OK) s = check_written(what, "out", args->out, a.rows, a.inner, a.cols);
    if (s != ZBPE_OK || !a.rows) return s;
    // in place each thread reads what it writes; otherwise a row that is loaded ahead could have been written already
    const Memory written(args->out, a.rows, a.inner, a.cols);
    const Memory logits(args->logits, a.rows, a.inner, a.cols);
    if (!(written == logits)) s = apart(what, "out", written, "the logits", logits);
    if (s == ZBPE_OK) s = apart_from_terms(what, "out", written, *args);
    if (s != ZBPE_OK) return s;
    OnDevice on;
    if ((s = on.go(device)) != ZBPE_OK) return s;
    return by_type(args->logits.dtype, [&](auto ti) {
        using T = decltype(ti);
        adjust_plan<T>(a.rows, a.cols, &a);
        const unsigned grid = grid_of(a.runs * a.slices);
        if (args->out.dtype == ZBPE_F32) adjust_kernel<T, float><<<grid, ADJUST_THREADS, 0, (hipStream_t)stream>>>(a);
        else adjust_kernel<T, T><<<grid, ADJUST_THREADS, 0, (hipStream_t)stream>>>(a);
        return launched(what);
    });
}

size_t zbpe_adjust_workspace(int64_t rows, int32_t cols) {
    if (rows < 1 || cols < 1 || cols > ZBPE_MAX_VOCAB) return 0;
    Adjust wide{}, narrow{};
    adjust_plan<float>(rows, cols, &wide);
    adjust_plan<f16>(rows, cols, &narrow);
    return (size_t)(wide.runs > narrow.runs ? wide.runs : narrow.runs) * (size_t)cols * sizeof(float);
}

zbpe_status zbpe_adjust_logits_grad(int device, void *stream, const zbpe_adjust *args, const zbpe_rows *grad_logits,
                                    float *grad_bias, float *grad_bias_values, void *workspace, size_t workspace_size) {
    const char *what = "zbpe_adjust_logits_grad";
    AdjustGrad g{};
    zbpe_status s = adjust_of(what, args, &g.a);
    if (s == ZBPE_OK) s = check_matrix(what, "the output's gradient", args->out, g.a.rows);
    if (s == ZBPE_OK && grad_logits) {
        if (grad_logits->dtype != args->logits.dtype) return refuse(ZBPE_INVALID_ARGUMENT, "%s: grad_logits has the type of the logits", what);
        s = check_written(what, "grad_logits", *grad_logits, g.a.rows, g.a.inner, g.a.cols);
        g.grad_logits = rows_of(*grad_logits);
        const Memory written(*grad_logits, g.a.rows, g.a.inner, g.a.cols);
        if (s == ZBPE_OK) s = apart(what, "grad_logits", written, "the logits", Memory(args->logits, g.a.rows, g.a.inner, g.a.cols));
        if (s == ZBPE_OK)
            s = apart(what, "grad_logits", written, "the output's gradient", Memory(args->out, g.a.rows, g.a.inner, g.a.cols));
        if (s == ZBPE_OK) s = apart_from_terms(what, "grad_logits", written, *args);
    }
    if (s != ZBPE_OK) return s;
    if (grad_bias && workspace_size < zbpe_adjust_workspace(g.a.rows, g.a.cols))
        return refuse(ZBPE_INVALID_ARGUMENT, "%s: a workspace of %zu bytes, %zu are needed", what, workspace_size, zbpe_adjust_workspace(g.a.rows, g.a.cols));
    if (grad_bias && !workspace && g.a.rows) return refuse(ZBPE_INVALID_ARGUMENT, "%s: no workspace", what);
    OnDevice on;
    if ((s = on.go(device)) != ZBPE_OK) return s;
    g.grad_bias_values = g.a.n_biases ? grad_bias_values : nullptr;
    g.sums = grad_bias ? (float *)workspace : nullptr;
    if (g.a.rows && (grad_logits || grad_bias || g.grad_bias_values)) {
        s = by_type(args->logits.dtype, [&](auto ti) {
            using T = decltype(ti);
            adjust_plan<T>(g.a.rows, g.a.cols, &g.a);
            const unsigned grid = grid_of(g.a.runs * g.a.slices);
            if (args->out.dtype == ZBPE_F32) adjust_grad_kernel<T, float><<<grid, ADJUST_THREADS, 0, (hipStream_t)stream>>>(g);
            else adjust_grad_kernel<T, T><<<grid, ADJUST_THREADS, 0, (hipStream_t)stream>>>(g);
            return launched(what);
        });
        if (s != ZBPE_OK) return s;
    }
    if (!grad_bias) return ZBPE_OK;
    adjust_bias_kernel<<<(unsigned)(g.a.cols + 63) / 64, 1024, 0, (hipStream_t)stream>>>(g.sums, g.a.runs, g.a.cols, grad_bias);
    return launched(what);
}

zbpe_status zbpe_draw_tokens(int device, void *stream, const zbpe_draw *p) {
    const char *what = "zbpe_draw_tokens";
    if (!p) return refuse(ZBPE_INVALID_ARGUMENT, "%s: no arguments", what);
    if (p->struct_size != sizeof(zbpe_draw)) return refuse(ZBPE_INVALID_ARGUMENT, "%s: arguments of another version", what);
    zbpe_status s = check_rows(what, p->rows, p->inner, p->cols);
    if (s == ZBPE_OK) s = check_matrix(what, "logits", p->logits, p->rows);
    if (s != ZBPE_OK || !p->rows) return s;
    if (!p->uniforms || !p->tokens) return refuse(ZBPE_INVALID_ARGUMENT, "%s: no uniforms, or no tokens", what);
    OnDevice on;
    if ((s = on.go(device)) != ZBPE_OK) return s;
    const Draw a{rows_of(p->logits), p->rows, p->inner, p->cols, p->uniforms, p->temperature, p->top_p, p->min_p, p->top_k, p->tokens, p->logprobs};
    return by_type(p->logits.dtype, [&](auto ti) {
        draw_launch<decltype(ti)>(a, (hipStream_t)stream);
        return launched(what);
    });
}

zbpe_status zbpe_token_logprobs(int device, void *stream, const zbpe_logprobs *args) {
    const char *what = "zbpe_token_logprobs";
    Logprobs a;
    zbpe_status s = logprobs_of(what, args, &a);
    if (s != ZBPE_OK || !a.rows) return s;
    if (!a.logprobs) return refuse(ZBPE_INVALID_ARGUMENT, "%s: no logprobs", what);
    OnDevice on;
    if ((s = on.go(device)) != ZBPE_OK) return s;
    return by_type(args->logits.dtype, [&](auto ti) {
        using T = decltype(ti);
        if (a.cols <= 2048) logprobs_kernel<T, 64><<<grid_of((a.rows + 3) / 4), 256, 0, (hipStream_t)stream>>>(a);
        else logprobs_kernel<T, 256><<<grid_of(a.rows), 256, 0, (hipStream_t)stream>>>(a);
        return launched(what);
    });
}

zbpe_status zbpe_token_logprobs_grad(int device, void *stream, const zbpe_logprobs *args, const float *grad,
                                     const zbpe_rows *grad_logits) {
    const char *what = "zbpe_token_logprobs_grad";
    Logprobs a;
    zbpe_status s = logprobs_of(what, args, &a);
    if (s != ZBPE_OK) return s;
    if (!grad_logits || grad_logits->dtype != args->logits.dtype) return refuse(ZBPE_INVALID_ARGUMENT, "%s: grad_logits has the type of the logits", what);
    if ((s = check_written(what, "grad_logits", *grad_logits, a.rows, a.inner, a.cols)) != ZBPE_OK || !a.rows) return s;
    if (!grad || !a.stats) return refuse(ZBPE_INVALID_ARGUMENT, "%s: no gradient, or no stats", what);
    const Memory written(*grad_logits, a.rows, a.inner, a.cols);
    const Memory logits(args->logits, a.rows, a.inner, a.cols);
    if (!(written == logits)) s = apart(what, "grad_logits", written, "the logits", logits);
    if (s == ZBPE_OK) s = apart(what, "grad_logits", written, "the tokens", Memory(a.tokens, (wide)a.rows * (args->tokens_dtype == ZBPE_I64 ? 8 : 4)));
    if (s == ZBPE_OK) s = apart(what, "grad_logits", written, "temperature", Memory(a.temperature, (wide)a.rows * 4));
    if (s == ZBPE_OK) s = apart(what, "grad_logits", written, "grad", Memory(grad, (wide)a.rows * 4));
    if (s == ZBPE_OK) s = apart(what, "grad_logits", written, "stats", Memory(a.stats, (wide)a.rows * 8));
    if (s != ZBPE_OK) return s;
    a.grad = grad;
    a.grad_logits = rows_of(*grad_logits);
    OnDevice on;
    if ((s = on.go(device)) != ZBPE_OK) return s;
    return by_type(args->logits.dtype, [&](auto ti) {
        using T = decltype(ti);
        const int each = 512 * Pack<T>::N, slices = (a.cols + each - 1) / each;
        logprobs_grad_kernel<T><<<dim3(grid_of(a.rows), (unsigned)slices), 256, 0, (hipStream_t)stream>>>(a);
        return launched(what);
    });
}

}  // extern "C"
