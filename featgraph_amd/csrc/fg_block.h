// Shared pieces of attention over selected blocks of keys: operand tiles of the matrix cores, the list of blocks that a tile of
// queries attends to, buckets of relative positions (included by .hip files only).
//
// Tiles.  v_mfma 16x16x32 multiplies a 16 x 32 by a 32 x 16 tile; with g = lane / 16 and c = lane % 16 a lane holds the eight elements
// k = 8 g .. 8 g + 7 of row c of the left and of column c of the right operand, and the rows 4 g .. 4 g + 3 of column c of the
// result.  The sum over k takes its terms in any order as long as both operands agree, so a result can be the right operand
// of the next product as it lies in the registers: its two row tiles give a lane the rows 4 g + i and 16 + 4 g + i, and the left
// operand is read in that order (`transposed`).  Scores are therefore formed with the softmax's rows as columns, (keys, queries)
// in the forward pass: every lane keeps the maximum and the sum of one query, and no result crosses lanes on its way into the second product.
// 32-bit elements take eight v_mfma 16x16x4 in the same places.
#pragma once

#include <hip/hip_runtime.h>

#include <cfloat>
#include <type_traits>

#include "fg_common.h"
#include "fg_device.h"

namespace fg {
namespace block {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Vec;
template <> struct Vec<__bf16> { typedef bf16x8 type; };
template <> struct Vec<_Float16> { typedef f16x8 type; };
template <> struct Vec<float> { typedef f32x8 type; };
template <typename T> using V8 = typename Vec<T>::type;

constexpr int kUnit = 32;              // keys (or query rows) of one step
constexpr int kWaves = 4;              // wavefronts of a workgroup
constexpr int kThreads = 64 * kWaves;
constexpr int kPad = 16;               // elements between staged rows: 16 rows' 32-byte pieces, and 128-bit writes, spread over the banks
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma(f32x8 a, f32x8 b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
}

template <typename T> __device__ __forceinline__ V8<T> load8(const T *p) { return *reinterpret_cast<const V8<T> *>(p); }
template <typename T> __device__ __forceinline__ V8<T> zero8() { return V8<T>{}; }

// Two results of four rows each (see above) as a right operand: rounded to the operands' type, to nearest.
template <typename T> __device__ __forceinline__ V8<T> pack(f32x4 a, f32x4 b) {
    V8<T> v;
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = (T)a[i]; v[4 + i] = (T)b[i]; }
    return v;
}

// The same, and what the rounding took, rounded itself (nothing in 32 bits).
template <typename T> __device__ __forceinline__ void split(f32x4 a, f32x4 b, V8<T> *high, V8<T> *low) {
    V8<T> v = pack<T>(a, b), w;
#pragma unroll
    for (int i = 0; i < 4; ++i) { w[i] = (T)(a[i] - (float)v[i]); w[4 + i] = (T)(b[i] - (float)v[4 + i]); }
    *high = v;
    *low = w;
}

// Elements (row, d0 + c) of a staged [32][D + kPad] tile for the rows 4 g + i and 16 + 4 g + i: columns of the tile as a left operand.
__device__ __forceinline__ s16x4 read_tr(const short *p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(p));
}
template <typename T, int D> __device__ __forceinline__ V8<T> transposed(const T *tile, int d0, int lane) {
    const int g = lane >> 4, c = lane & 15;
    constexpr int S = D + kPad;
    V8<T> v;
    if constexpr (sizeof(T) == 2) {
        // of each 16 lanes, lane c brings the address of row c / 4, columns 4 (c % 4) .. + 3, and takes column c of the four rows
        const short *p = reinterpret_cast<const short *>(tile) + (4 * g + (c >> 2)) * S + d0 + 4 * (c & 3);
        const s16x4 lo = read_tr(p), hi = read_tr(p + 16 * S);
        v = __builtin_bit_cast(V8<T>, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[i] = tile[(4 * g + i) * S + d0 + c]; v[4 + i] = tile[(16 + 4 * g + i) * S + d0 + c]; }
    }
    return v;
}

// acc + a (b + low), where b's element is a factor only if its bit in `seen` is set, with what infinities and NaN in a give: a masked pair adds
// nothing whatever a holds.  `low` is what rounding took from b (split), or 0.  Their places are marked by further products of ones and
// zeros.  For tiles in which the plain product left something that is not finite; everything else takes mma() alone.
template <typename T> __device__ __forceinline__ f32x4 mma_masked(V8<T> a, V8<T> b, V8<T> low, unsigned seen, f32x4 acc) {
    V8<T> fin, ap, an, ax, bad, bs, bp, bn, bz;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float x = (float)a[i], y = (float)b[i];
        const bool s = (seen >> i) & 1u, inf = fabsf(x) == __builtin_inff(), nan = x != x;
        fin[i] = inf || nan ? (T)0.f : a[i];
        ap[i] = (T)(inf && x > 0 ? 1.f : 0.f); an[i] = (T)(inf && x < 0 ? 1.f : 0.f);
        ax[i] = (T)(nan ? 1.f : 0.f);          bad[i] = (T)(inf || nan ? 1.f : 0.f);
        low[i] = fabsf(y) < __builtin_inff() ? low[i] : (T)0.f;
        bs[i] = (T)(s ? 1.f : 0.f);            bz[i] = (T)(s && !(y > 0 || y < 0) ? 1.f : 0.f);
        bp[i] = (T)(s && y > 0 ? 1.f : 0.f);   bn[i] = (T)(s && y < 0 ? 1.f : 0.f);
    }
    const f32x4 none = {0.f, 0.f, 0.f, 0.f};
    acc = mma(fin, b, acc);
    if (sizeof(T) == 2) acc = mma(fin, low, acc);
    const f32x4 pos = mma(ap, bp, mma(an, bn, none)), neg = mma(ap, bn, mma(an, bp, none)), no = mma(bad, bz, mma(ax, bs, none));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (pos[i] > 0.f) acc[i] += __builtin_inff();
        if (neg[i] > 0.f) acc[i] -= __builtin_inff();
        if (no[i] > 0.f) acc[i] = __builtin_nanf("");
    }
    return acc;
}

__device__ __forceinline__ bool not_finite(f32x4 v) {
    // x - x is 0 for a number, NaN otherwise
    const float t = (v[0] - v[0]) + (v[1] - v[1]) + (v[2] - v[2]) + (v[3] - v[3]);
    return t != t;
}

// What rounding took from a result is at most half of its last place.  float16 has no numbers for that below 2^-24, and few bits for it below 2^-3: it
// is stored 2^11 times as large, of the result's own size.
template <typename T> constexpr float kRestScale = std::is_same<T, _Float16>::value ? 2048.f : 1.f;

// Four consecutive elements of a result, rounded to its type, and what the rounding took where that is wanted.
template <typename T> __device__ __forceinline__ void store_row(T *out, T *rest, int64_t at, f32x4 v) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    T4 x, y;
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[i] = (T)v[i]; y[i] = (T)((v[i] - (float)x[i]) * kRestScale<T>); }
    *reinterpret_cast<T4 *>(out + at) = x;
    if (rest) *reinterpret_cast<T4 *>(rest + at) = y;
}

// The largest of eight numbers (NaN only if all are).  Written out: of products of the matrix cores the compiler takes every operand's
// maximum with itself first, which doubles the instructions.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm volatile("v_max3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));        // volatile: not moved behind a branch
    return d;
}
__device__ __forceinline__ float largest(f32x4 a, f32x4 b) { return max3(max3(max3(a[0], a[1], a[2]), a[3], b[0]), max3(b[1], b[2], b[3]), b[3]); }
// The largest of lanes l, l ^ 16, l ^ 32, l ^ 48; every lane gets it.
__device__ __forceinline__ float largest_of_rows(float v) {
    float w = v;
    swap_halves(v, w);
    float x = max3(v, w, w), y = x;
    swap_rows(x, y);
    return max3(x, y, y);
}

struct Strides { int64_t batch, row, head; };    // in elements

// What every kernel of the operator takes.
struct Problem {
    int batch, queries, keys, heads, kv_heads, group, block_shift, blocks, topk, causal;
    float scale, scale2;                         // the scores' scale, and that times log2(e): exponentials are powers of two
    const void *q, *k, *v, *bias;
    Strides qs, ks, vs;
    const int32_t *list, *lengths, *q_lengths;
    int n_buckets, low, high;                    // bucket 0 up to `low`, the last one from `high`
    int32_t bounds[63];
};

__device__ __forceinline__ int key_count(const Problem &p, int b) {
    return p.lengths ? min(max(p.lengths[b], 0), p.keys) : p.keys;
}
__device__ __forceinline__ int query_count(const Problem &p, int b) {
    return p.q_lengths ? min(max(p.q_lengths[b], 0), p.queries) : p.queries;
}

// Tokens of one tile of 16 rows (all the heads that share a key head), so that a lane's column has the same head in every tile.
__host__ __device__ __forceinline__ int tile_tokens(int group) { return 16 / group; }

// Which of a sequence's groups of tiles a workgroup takes: the last tokens first where they are causal, for they have the most blocks to
// choose from and the longest lists (8,192 tokens, 32 / 8 heads 450 -> 408 us, dQ of 2 x 4,096 tokens 319 -> 274).
__device__ __forceinline__ int group_of(const Problem &p, int i, int n) { return p.causal ? n - 1 - i : i; }

// The blocks that some tiles of queries attend to, window by window: block ids (within the window) in ascending order and, for each, the tokens
// that selected it: 16 bits for every tile, bit t for its token t.  An index that is negative, behind the keys, behind the query or named
// twice counts for nothing more.
template <int TILES, int WINDOW>
struct List {
    static constexpr int kWords = (TILES + 3) / 4, kWidth = WINDOW;
    unsigned long long bits[WINDOW][kWords];
    uint16_t id[WINDOW];
    int sums[kWaves];
};

// Builds the list for blocks [first, first + width) and the tokens of `tiles` tiles from t0 on, of sequence b, key head h; returns its length.  For
// all threads of the workgroup.
template <int TILES, int WINDOW>
__device__ __forceinline__ int build_list(List<TILES, WINDOW> &l, const Problem &p, int b, int h, int t0, int q_len, int k_len, int first, int width) {
    constexpr int WORDS = List<TILES, WINDOW>::kWords;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, tpt = tile_tokens(p.group);
    __syncthreads();                                   // of the last window
    for (int i = tid; i < width * WORDS; i += kThreads) l.bits[0][i] = 0;
    __syncthreads();
    const int there = min(TILES * tpt, q_len - t0), offset = k_len - q_len;
    const int64_t row = (int64_t)p.kv_heads * p.topk;
    const int32_t *src = p.list + ((int64_t)b * p.queries + t0) * row + (int64_t)h * p.topk;
    for (int e = tid; e < there * p.topk; e += kThreads) {
        const int t = e / p.topk, blk = src[t * row + (e - t * p.topk)], at = blk - first;
        if (at < 0 || at >= width) continue;           // blk < p.blocks, as first + width is
        const int key = blk << p.block_shift, tile = t / tpt;
        if (key < k_len && (!p.causal || key <= offset + t0 + t)) atomicOr(&l.bits[at][tile >> 2], 1ull << ((tile & 3) * 16 + t - tile * tpt));
    }
    __syncthreads();
    constexpr int C = (WINDOW + kThreads - 1) / kThreads;
    const int per = (width + kThreads - 1) / kThreads; // consecutive blocks of a thread, C at most
    unsigned long long mine[C][WORDS];
    int count = 0;
#pragma unroll
    for (int i = 0; i < C; ++i) {
        const int at = tid * per + i;
        unsigned long long any = 0;
#pragma unroll
        for (int w = 0; w < WORDS; ++w) any |= mine[i][w] = i < per && at < width ? l.bits[at][w] : 0;
        count += any != 0;
    }
    int upto = count;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(upto, d);
        if (lane >= d) upto += o;
    }
    if (lane == 63) l.sums[wave] = upto;
    __syncthreads();
    int before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        before += w < wave ? l.sums[w] : 0;
        total += l.sums[w];
    }
    int at = before + upto - count;
#pragma unroll
    for (int i = 0; i < C; ++i) {
        unsigned long long any = 0;
#pragma unroll
        for (int w = 0; w < WORDS; ++w) any |= mine[i][w];
        if (any) {
#pragma unroll
            for (int w = 0; w < WORDS; ++w) l.bits[at][w] = mine[i][w];
            l.id[at++] = (uint16_t)(tid * per + i);
        }
    }
    __syncthreads();
    return total;
}

// 64 keys of one operand on their way into LDS: 128-bit words of a workgroup's threads, rows `stride` elements apart there.  The two halves are
// units of 32 keys, k0 .. and k1 ..; rows behind the last key read it again, so that what a padded cache holds there is never touched.
template <typename T, int D> struct Stage {
    static constexpr int EPC = 16 / sizeof(T), CPR = D / EPC, RPL = kThreads / CPR, N = 2 * kUnit / RPL;
    u32x4 word[N];
    __device__ __forceinline__ void fetch(const T *base, int64_t row_stride, int k0, int k1, int k_len) {
        const int r0 = threadIdx.x / CPR, col = threadIdx.x % CPR * EPC;
        if (max(k0, k1) + kUnit <= k_len) {            // the rows' distances are the same in every step
            const T *own = base + r0 * row_stride + col;
            if constexpr (RPL <= kUnit) {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    word[i] = *reinterpret_cast<const u32x4 *>(own + ((i * RPL < kUnit ? k0 : k1 - kUnit) + i * RPL) * row_stride);
            } else {
                word[0] = *reinterpret_cast<const u32x4 *>(own + (r0 < kUnit ? k0 : k1 - kUnit) * row_stride);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int r = i * RPL + r0;
                word[i] = *reinterpret_cast<const u32x4 *>(base + min((r < kUnit ? k0 : k1 - kUnit) + r, k_len - 1) * row_stride + col);
            }
        }
    }
    __device__ __forceinline__ void store(T *tile, int stride) const {
        const int r0 = threadIdx.x / CPR, col = threadIdx.x % CPR * EPC;
#pragma unroll
        for (int i = 0; i < N; ++i) *reinterpret_cast<u32x4 *>(tile + (i * RPL + r0) * stride + col) = word[i];
    }
};

// The bias by relative position, in LDS: the bucket of every distance from `low` to `high`, and every bucket's bias for the heads of one
// group, times log2(e).
constexpr int kSpan = 4096;            // most distances between the first bound and the last
struct Buckets {
    const uint8_t *of;
    const float *bias;                 // [n_buckets][group]
    int low, high, group;
    __device__ __forceinline__ int at(int distance) const { return of[min(max(distance, low), high) - low]; }
    __device__ __forceinline__ float value(int bucket, int head) const { return bias[bucket * group + head]; }
};
__host__ __device__ __forceinline__ size_t buckets_bytes(int n_buckets, int low, int high, int group) {
    return n_buckets ? (size_t)((high - low + 1 + 15) & ~15) + (size_t)n_buckets * group * sizeof(float) : 0;
}
template <typename T>
__device__ __forceinline__ Buckets load_buckets(const Problem &p, int h, unsigned char *lds) {
    const int span = p.high - p.low + 1;
    float *bias = reinterpret_cast<float *>(lds + ((span + 15) & ~15));
    for (int i = threadIdx.x; i < span; i += kThreads) {
        int n = 0;
        for (int j = 0; j + 1 < p.n_buckets; ++j) n += p.bounds[j] <= p.low + i;
        lds[i] = (uint8_t)n;
    }
    const T *src = static_cast<const T *>(p.bias);
    for (int i = threadIdx.x; i < p.n_buckets * p.group; i += kThreads) {
        const int n = i / p.group;
        // the type's lowest value, used as a mask, stays finite: rows that see nothing else have a softmax
        const float x = (float)src[(int64_t)n * p.heads + h * p.group + (i - n * p.group)], y = x * kLog2e;
        bias[i] = fabsf(x) < __builtin_inff() ? fminf(fmaxf(y, -FLT_MAX), FLT_MAX) : y;
    }
    return Buckets{lds, bias, p.low, p.high, p.group};
}

// Fills a Problem from the C interface's arguments; FG_OK or an error with its message.
int problem_of(const fg_block_attention_args *a, Problem *p);
// A dense array that the kernels access `bytes` at a time; null is fine.
int aligned(const char *name, const void *ptr, int bytes);
// A strided operand: dense heads, every one of them at a 16-byte address.
int strides_of(const char *name, const void *ptr, const int64_t *stride, int size, Strides *s);
}  // namespace block
}  // namespace fg
