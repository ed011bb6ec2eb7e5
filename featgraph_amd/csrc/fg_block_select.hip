// Choosing blocks of keys by a cheap score: the keys' mean over each block, and for every query the blocks with the highest product of
// that mean and the sum of the queries that share the key head.
//
// fg_block_pool reads the keys once (HBM bound: 16,384 keys of 8 heads of 128 7.6 us, 4.4 TB/s).  fg_block_select forms the scores of 16 queries on the matrix cores, keeps them in LDS (they
// are never written to memory) and lets one wavefront at a time find a query's topk.  Two blocks whose scores the 32-bit sums
// cannot tell apart would come out in an order that depends on the order of the sums, and with them the whole attention of a
// query; so a second product bounds the error, and blocks within it of the topk-th score are compared again in 64 bits.  Finding the topk is
// what takes the time (16,384 queries, 32 / 8 heads of 128, up to 256 blocks: 110 us, of which the queries' bytes would take 30 and the
// products 7): vector and scalar instructions of counting, in one wavefront per query.
#include <algorithm>
#include <type_traits>

#include "fg_block.h"

namespace fg {
namespace block {

namespace {

// A 64-bit number in the operands' type, by way of 32 bits as tensors are converted.  The compiler would make the two steps one and round
// some numbers next to the middle of two of the type the other way.
template <typename T> __device__ __forceinline__ T narrow(double x) {
    float f = (float)x;
    asm volatile("" : "+v"(f));
    return (T)f;
}

// One workgroup per block of keys and key head.  Sums in 64 bits, whatever their order; the mean is rounded to 32 bits and then to the type, as tensors
// are converted.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void pool_kernel(const T *k, Strides ks, const int32_t *lengths, T *pooled, int keys, int kv_heads, int block, int blocks) {
    constexpr int EPC = 16 / sizeof(T), CPR = D / EPC, ROWS = kThreads / CPR;
    __shared__ double sums[ROWS][D];
    const int n = blockIdx.x % blocks, pair = blockIdx.x / blocks, b = pair / kv_heads, h = pair - b * kv_heads;
    const int k_len = lengths ? min(max(lengths[b], 0), keys) : keys;
    const int first = n * block, count = min(block, max(k_len - first, 0));
    const int chunk = threadIdx.x % CPR, row = threadIdx.x / CPR;
    const T *src = k + b * ks.batch + h * ks.head + (int64_t)first * ks.row + chunk * EPC;
    typedef T Chunk __attribute__((ext_vector_type(EPC)));
    double acc[EPC];
#pragma unroll
    for (int i = 0; i < EPC; ++i) acc[i] = 0;
    for (int r = row; r < count; r += ROWS) {
        const Chunk x = *reinterpret_cast<const Chunk *>(src + (int64_t)r * ks.row);
#pragma unroll
        for (int i = 0; i < EPC; ++i) acc[i] += (double)(float)x[i];
    }
#pragma unroll
    for (int i = 0; i < EPC; ++i) sums[row][chunk * EPC + i] = acc[i];
    __syncthreads();
    for (int d = threadIdx.x; d < D; d += kThreads) {
        double total = 0;
        for (int r = 0; r < ROWS; ++r) total += sums[r][d];
        pooled[((int64_t)pair * blocks + n) * D + d] = narrow<T>(count ? total / count : 0.0);
    }
}

// Numbers as unsigned integers of the same order; NaN as -inf.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x != x ? -__builtin_inff() : x);
    return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_ordered(uint32_t u) { return __uint_as_float(u >> 31 ? u & 0x7fffffffu : ~u); }
__device__ __forceinline__ unsigned long long ordered(double x) {
    const unsigned long long u = (unsigned long long)__double_as_longlong(x != x ? -__builtin_inf() : x + 0.0);    // -0 is 0
    return u >> 63 ? ~u : u | (1ull << 63);
}

// Where the `count` largest of the wavefront's keys (R in each lane) begin: a value that exactly `count` of them reach, or, where equal keys
// leave none, the largest value that at least as many reach.  From the top bit down, four bits between looks at whether it is
// found (a look at every bit costs more than it saves: 256 blocks per query, 16,384 queries 117 us, 512 blocks, one query 20.7; four 108
// and 15).
template <int R, typename K>
__device__ __forceinline__ K cut_off(const K (&key)[R], int count, bool *exactly) {
    K at = 0;
    int reached = -1;
    for (int bit = 8 * sizeof(K) - 1; bit >= 0 && reached != count; bit -= 4) {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const K trial = at | ((K)1 << (bit - b));
            int n = 0;
#pragma unroll
            for (int r = 0; r < R; ++r) n += __popcll(__ballot(key[r] >= trial));
            at = n >= count ? trial : at;
            reached = n >= count ? n : reached;
        }
    }
    *exactly = reached == count;
    return at;
}

constexpr int kTokens = 16;
constexpr int kMaxBlocks = 2048;

template <typename T, int D, int R>
__global__ __launch_bounds__(kThreads) void select_kernel(const T *q, Strides qs, const T *pooled, const int32_t *lengths, const int32_t *q_lengths,
                                                          int32_t *out, int queries, int keys, int kv_heads, int group, int block_shift, int blocks,
                                                          int topk, int causal, int keep_first, int keep_last, int n_tiles, int stride) {
    constexpr int DC = D / 32;
    __shared__ __align__(16) T summed[kTokens][D + 8];
    __shared__ float mass[kWaves][kTokens];
    __shared__ int close_ids[kWaves][16];
    extern __shared__ __align__(16) float scores[];        // [kTokens][stride]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, c = lane & 15;
    const int unit = xcd_contiguous_block(), pair = unit / n_tiles, t0 = (unit - pair * n_tiles) * kTokens, b = pair / kv_heads, h = pair - b * kv_heads;
    const int k_len = lengths ? min(max(lengths[b], 0), keys) : keys, q_len = q_lengths ? min(max(q_lengths[b], 0), queries) : queries;
    const int offset = k_len - q_len;
    // candidates of a query are the blocks 0 .. candidates() - 1
    auto candidates = [&](int t) {
        const int last = causal ? min(offset + t, k_len - 1) : k_len - 1;
        return t < q_len && last >= 0 ? (last >> block_shift) + 1 : 0;
    };
    const int most = candidates(min(t0 + kTokens, q_len) - 1);
    const T *means = pooled + (int64_t)pair * blocks * D;

    for (int dc = wave; dc < DC; dc += kWaves) {
        const int t = t0 + c;
        double acc[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = 0;
        if (t < q_len) {
            const T *src = q + b * qs.batch + (int64_t)t * qs.row + (int64_t)h * group * qs.head + dc * 32 + 8 * g;
            for (int x = 0; x < group; ++x) {
                const V8<T> v = load8(src + x * qs.head);
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[i] += (double)(float)v[i];
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) summed[c][dc * 32 + 8 * g + i] = narrow<T>(acc[i]);
    }
    __syncthreads();
    V8<T> qf[DC], qa[DC];
    auto magnitude = [](V8<T> v) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (T)fabsf((float)v[i]);
        return v;
    };
#pragma unroll
    for (int dc = 0; dc < DC; ++dc) { qf[dc] = load8(&summed[c][dc * 32 + 8 * g]); qa[dc] = magnitude(qf[dc]); }
    float sum_abs = 0.f;
    for (int j0 = wave * 16; j0 < most; j0 += 16 * kWaves) {
        const T *src = means + (int64_t)min(j0 + c, blocks - 1) * D + 8 * g;
        f32x4 s = {0.f, 0.f, 0.f, 0.f}, a = s;
#pragma unroll
        for (int dc = 0; dc < DC; ++dc) {
            const V8<T> x = load8(src + dc * 32);
            s = mma(x, qf[dc], s);
            a = mma(magnitude(x), qa[dc], a);
        }
        *reinterpret_cast<f32x4 *>(scores + c * stride + j0 + 4 * g) = s;
        sum_abs = fmaxf(sum_abs, fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3])));
    }
    sum_abs = rows_max(sum_abs);
    if (g == 0) mass[wave][c] = sum_abs;
    __syncthreads();

    for (int i = 0; i < kTokens / kWaves; ++i) {
        const int tt = wave * (kTokens / kWaves) + i, t = t0 + tt;
        if (t >= queries) break;
        int32_t *dst = out + (((int64_t)b * queries + t) * kv_heads + h) * topk;
        const int n = candidates(t);
        if (n <= topk) {
            for (int j = lane; j < topk; j += 64) dst[j] = j < n ? j : -1;
            continue;
        }
        // key 0: no candidate; all ones: taken for certain
        uint32_t key[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int j = r * 64 + lane;
            key[r] = j >= n ? 0u : j < keep_first || j >= n - keep_last ? ~0u : ordered(scores[tt * stride + j]);
        }
        bool exactly;
        const uint32_t cut = cut_off<R, uint32_t>(key, topk, &exactly);
        // |32-bit sum of D products - exact| <= D u sum |products|, u = 2^-23 should the matrix cores cut instead of round; twice
        // that, for the bound is a sum of the same kind.  A block two errors above the cut beats every block below it, exactly, and one
        // two errors below is beaten by the topk above it.
        const float err = (D + 8) * 2.4e-7f * fmaxf(fmaxf(mass[0][tt], mass[1][tt]), fmaxf(mass[2][tt], mass[3][tt])) + 1e-34f;
        const float at = of_ordered(cut), high = at + 2 * err, low = at - 2 * err;
        unsigned in = 0, maybe = 0;
        int n_in = 0, n_maybe = 0;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float s = of_ordered(key[r]);
            const bool sure = key[r] == ~0u || (key[r] && s > high), close = key[r] && !sure && !(s < low);
            in |= (unsigned)sure << r;
            maybe |= (unsigned)close << r;
            n_in += __popcll(__ballot(sure));
            n_maybe += __popcll(__ballot(close));
        }
        const int need = topk - n_in;
        if (need == n_maybe) {
            in |= maybe;
        } else if (need > 0 && n_maybe <= 16) {
            // mostly two or three of them: a quarter of a product to a lane
            int base = 0;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const unsigned long long all = __ballot((maybe >> r) & 1);
                if ((maybe >> r) & 1) close_ids[wave][base + __popcll(all & ((1ull << lane) - 1))] = r * 64 + lane;
                base += __popcll(all);
            }
            wave_lds_sync();
            const int id = c < n_maybe ? close_ids[wave][c] : 0;
            const T *src = means + (int64_t)id * D + g * (D / 4);
            double dot = 0;
#pragma unroll
            for (int d = 0; d < D / 4; d += 8) {
                const V8<T> x = load8(src + d), y = load8(&summed[tt][g * (D / 4) + d]);
#pragma unroll
                for (int e = 0; e < 8; ++e) dot += (double)(float)x[e] * (double)(float)y[e];
            }
            dot += __shfl_xor(dot, 16);
            dot += __shfl_xor(dot, 32);
            const unsigned long long fine[1] = {g == 0 && c < n_maybe ? ordered(dot) : 0};
            unsigned long long edge = cut_off<1, unsigned long long>(fine, need, &exactly);
            edge -= exactly;                       // `need` of them are above it, or those above and some that are equal
            const unsigned long long above = __ballot(fine[0] > edge);
            unsigned long long same = exactly ? 0 : __ballot(fine[0] && fine[0] == edge), taken = above;
            for (int left = need - __popcll(above); left > 0; --left, same &= same - 1) taken |= same & -same;     // the lowest ids
            for (; taken; taken &= taken - 1) {
                const int one = __shfl(id, __builtin_ctzll(taken));
                in |= lane == (one & 63) ? 1u << (one >> 6) : 0u;
            }
            wave_lds_sync();
        } else if (need > 0) {
            unsigned long long fine[R];
#pragma unroll
            for (int r = 0; r < R; ++r) fine[r] = 0;
#pragma unroll 1
            for (int r = 0; r * 64 < n; ++r) {
                const bool look = (maybe >> r) & 1;
                if (!__ballot(look)) continue;
                const T *src = means + (int64_t)(look ? r * 64 + lane : 0) * D;
                double dot = 0;
#pragma unroll 4
                for (int d = 0; d < D; d += 8) {
                    const V8<T> x = load8(src + d), y = load8(&summed[tt][d]);
#pragma unroll
                    for (int e = 0; e < 8; ++e) dot += (double)(float)x[e] * (double)(float)y[e];
                }
                const unsigned long long v = look ? ordered(dot) : 0;
#pragma unroll
                for (int x = 0; x < R; ++x) fine[x] = x == r ? v : fine[x];
            }
            unsigned long long edge = cut_off<R, unsigned long long>(fine, need, &exactly);
            edge -= exactly;                       // `need` of them are above it, or those above and some that are equal
            int above = 0;
#pragma unroll
            for (int r = 0; r < R; ++r) above += __popcll(__ballot(fine[r] > edge));
            int equal = need - above;              // of those at the edge, the lowest ids
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const unsigned long long same = __ballot(fine[r] == edge && ((maybe >> r) & 1));
                const bool take = fine[r] > edge || (((same >> lane) & 1) && __popcll(same & ((1ull << lane) - 1)) < equal);
                equal -= min(equal, (int)__popcll(same));
                in |= (unsigned)take << r;
            }
        }
        int base = 0;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const unsigned long long all = __ballot((in >> r) & 1);
            const int place = base + __popcll(all & ((1ull << lane) - 1));
            if ((in >> r) & 1) dst[place] = r * 64 + lane;
            base += __popcll(all);
        }
    }
}

template <typename T, int D>
int launch_pool(const void *k, Strides ks, const int32_t *lengths, void *pooled, int pairs, int keys, int kv_heads, int block, hipStream_t stream) {
    const int blocks = (keys + block - 1) / block;
    const int64_t grid = (int64_t)pairs * blocks;
    if (grid >= (1ll << 31)) return fail(FG_ERR_SHAPE, "block pool: %lld workgroups do not fit a launch", (long long)grid);
    pool_kernel<T, D><<<dim3((unsigned)grid), dim3(kThreads), 0, stream>>>(static_cast<const T *>(k), ks, lengths, static_cast<T *>(pooled), keys, kv_heads, block, blocks);
    FG_HIP_TRY(hipGetLastError());
    return FG_OK;
}

struct Choice {
    const void *q, *pooled;
    Strides qs;
    const int32_t *lengths, *q_lengths;
    int32_t *out;
    int batch, queries, keys, kv_heads, group, block, topk, causal, keep_first, keep_last;
};

template <typename T, int D, int R>
int launch_select_r(const Choice &c, int blocks, hipStream_t stream) {
    const int n_tiles = (c.queries + kTokens - 1) / kTokens, stride = ((blocks + 15) & ~15) + 4;
    const size_t lds = (size_t)kTokens * stride * sizeof(float);
    const int64_t grid = (int64_t)c.batch * c.kv_heads * n_tiles;
    if (grid >= (1ll << 31)) return fail(FG_ERR_SHAPE, "block select: %lld workgroups do not fit a launch", (long long)grid);
    select_kernel<T, D, R><<<dim3((unsigned)grid), dim3(kThreads), lds, stream>>>(
        static_cast<const T *>(c.q), c.qs, static_cast<const T *>(c.pooled), c.lengths, c.q_lengths, c.out, c.queries, c.keys, c.kv_heads, c.group,
        31 - __builtin_clz(c.block), blocks, c.topk, c.causal, c.keep_first, c.keep_last, n_tiles, stride);
    FG_HIP_TRY(hipGetLastError());
    return FG_OK;
}
template <typename T, int D>
int launch_select(const Choice &c, hipStream_t stream) {
    const int blocks = (c.keys + c.block - 1) / c.block;
    // Registers for a query's scores, one per 64 blocks, of four kinds.  2,048 queries, 32 / 8 heads of 128: 128 blocks 20 us, 130 23, 256 29,
    // 260 36, 512 45, 513 130, 1,024 147, 2,048 297: the last kind is for caches beyond 512 blocks, and those between pay for its 32 registers.
    return blocks <= 128 ? launch_select_r<T, D, 2>(c, blocks, stream) : blocks <= 256 ? launch_select_r<T, D, 4>(c, blocks, stream) : blocks <= 512 ? launch_select_r<T, D, 8>(c, blocks, stream)
                                                                                      : launch_select_r<T, D, 32>(c, blocks, stream);
}

// f(type, head length as constants)
template <typename F> int by_type(int type, int head_len, F f) {
    auto by_length = [&](auto x) {
        switch (head_len) {
        case 32: return f(x, std::integral_constant<int, 32>{});
        case 64: return f(x, std::integral_constant<int, 64>{});
        default: return f(x, std::integral_constant<int, 128>{});
        }
    };
    return type == FG_TYPE_F32 ? by_length(0.f) : type == FG_TYPE_F16 ? by_length((_Float16)0.f) : by_length((__bf16)0.f);
}

int check_common(const char *what, int type, const void *x, const int64_t *stride, int batch, int keys, int kv_heads, int head_len, int block) {
    if (type != FG_TYPE_F32 && type != FG_TYPE_F16 && type != FG_TYPE_BF16) return fail(FG_ERR_ARG, "%s: unknown type %d", what, type);
    if (batch < 0 || keys < 0 || kv_heads < 1 || !stride) return fail(FG_ERR_ARG, "%s: negative sizes, no heads, or a null pointer", what);
    if (keys > (1 << 30)) return fail(FG_ERR_SHAPE, "%s: more than 2^30 keys", what);
    if (head_len != 32 && head_len != 64 && head_len != 128) return fail(FG_ERR_SHAPE, "%s: heads of 32, 64 or 128 elements, got %d", what, head_len);
    if (block != 32 && block != 64 && block != 128 && block != 256) return fail(FG_ERR_SHAPE, "%s: blocks of 32, 64, 128 or 256 keys, got %d", what, block);
    const int64_t per = type == FG_TYPE_F32 ? 4 : 8;
    if (reinterpret_cast<uintptr_t>(x) % 16 || stride[0] % per || stride[1] % per || stride[2] % per)
        return fail(FG_ERR_ARG, "%s: the operand and its strides have to be multiples of 16 bytes", what);
    return FG_OK;
}
}  // namespace
}  // namespace block
}  // namespace fg

extern "C" int fg_block_pool(int type, const void *k_dev, const int64_t *k_strides, const int32_t *lengths_dev, void *pooled_dev, int batch, int keys,
                             int kv_heads, int head_len, int block, void *stream) {
    using namespace fg::block;
    if (int rc = check_common("block pool", type, k_dev, k_strides, batch, keys, kv_heads, head_len, block)) return rc;
    if (batch == 0 || keys == 0) return FG_OK;
    if (!k_dev || !pooled_dev) return fg::fail(FG_ERR_ARG, "block pool: null pointer");
    const Strides ks{k_strides[0], k_strides[1], k_strides[2]};
    return by_type(type, head_len, [&](auto x, auto d) {
        return launch_pool<decltype(x), decltype(d)::value>(k_dev, ks, lengths_dev, pooled_dev, batch * kv_heads, keys, kv_heads, block, static_cast<hipStream_t>(stream));
    });
}

extern "C" int fg_block_select(int type, const void *q_dev, const int64_t *q_strides, const void *pooled_dev, const int32_t *lengths_dev,
                               const int32_t *q_lengths_dev, int32_t *blocks_dev, int batch, int queries, int keys, int heads, int kv_heads, int head_len,
                               int block, int topk, int causal, int keep_first, int keep_last, void *stream) {
    using namespace fg::block;
    if (int rc = check_common("block select", type, q_dev, q_strides, batch, keys, kv_heads, head_len, block)) return rc;
    if (queries < 0 || queries > (1 << 30) || topk < 1 || keep_first < 0 || keep_last < 0 || keep_first > topk - keep_last)
        return fg::fail(FG_ERR_ARG, "block select: %d queries, %d blocks of which the first %d and the last %d are kept", queries, topk, keep_first, keep_last);
    if (heads < 1 || heads % kv_heads) return fg::fail(FG_ERR_SHAPE, "block select: %d heads over %d key heads", heads, kv_heads);
    if ((keys + block - 1) / block > kMaxBlocks) return fg::fail(FG_ERR_SHAPE, "block select: %d keys are more than %d blocks of %d", keys, kMaxBlocks, block);
    if (batch == 0 || queries == 0) return FG_OK;
    if (!q_dev || !blocks_dev || (keys && !pooled_dev)) return fg::fail(FG_ERR_ARG, "block select: null pointer");
    if (reinterpret_cast<uintptr_t>(pooled_dev) % 16) return fg::fail(FG_ERR_ARG, "block select: the pooled keys have to stand at a multiple of 16 bytes");
    const Choice c{q_dev, pooled_dev, Strides{q_strides[0], q_strides[1], q_strides[2]}, lengths_dev, q_lengths_dev, blocks_dev,
                   batch, queries, keys, kv_heads, heads / kv_heads, block, topk, causal != 0, keep_first, keep_last};
    return by_type(type, head_len, [&](auto x, auto d) { return launch_select<decltype(x), decltype(d)::value>(c, static_cast<hipStream_t>(stream)); });
}
