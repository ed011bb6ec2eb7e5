// Softmax attention of a few queries over a cache of 4 or 8 bits, whole or the blocks that a list names:
//   out[i, h] = sum_j p_ij V[j, g],  p_i = softmax over the visible keys j of  scale <Q[i, h], K[j, g]>
// with g = h / group, pos_i = k_len - q_len + i, and j visible to i where j < k_len, (causal) j <= pos_i and, where there is a list, floor(j / block)
// is in i's list for g.  No visible key: 0.
//
// Every value of the cache is a bfloat16, so that products with it are bfloat16 products of the matrix cores, exact up to the sums in 32
// bits, whatever type the queries have: a float16 is the sum of two bfloat16, a number of 32 bits of three.  Powers are taken apart the
// same way, each rounded to nearest: into two parts for 16-bit results (up to 2^-17 of a power is lost) and three for 32-bit ones (nothing is).
// Rows of one token's heads and of neighbouring tokens make tiles of 16, RT of them a workgroup.  Its four wavefronts deal the keys out among themselves, 32 at a
// time, and where there are too few workgroups for the card so do several workgroups, whose sums are joined after.  A
// lane's keys come from memory as operands lie in registers (the sum over a head's elements takes them in any order), values go
// through LDS as bfloat16 to be read by columns; the next step is under way while one is worked on.
// Values that are no numbers are taken as 0 and marked; the marks of the keys that a row sees make its result NaN.  (Keys that are none, and queries that
// are not finite, make scores of their own rows alone.)
//
// What bounds it.  32 requests of 32,768 keys of 8 heads x 128 in 4 bits, one token of 32 heads each (1.14 GB): 196 us, 5.8 TB/s, above the rate of a large copy (5.1),
// for it only reads; two wavefronts a SIMD, which is what the rule for shares launches there, keep 8.7 KB each SIMD on their way. With a sweep of its own for values that are not finite in
// the same kernel it took 276 registers and 353 us.  One request of 2,048 keys x 8 heads x 64: 7.6 us captured, of which some 3.5 are the joining launch and the rest the chain
// length, keys, softmax, joining. Many rows, 64 tokens over 16,384 keys of 8 x 128 in 8 bits: 42 us, 410 TFLOP/s counted once; with two tiles of rows two
// wavefronts fit a SIMD, each of which issues a vector instruction or a product in 31 % of its cycles and waits in 26 % (348 vector instructions a step, 52 of them products).  (Four
// wavefronts that share the widened keys through LDS and take two tiles each wait for one another: 46 us, and 134 where this takes 111, 512 tokens over 8,192 keys.)
#include <algorithm>
#include <type_traits>

#include "fg_cache.h"

namespace fg {
namespace cache {

namespace {

using namespace block;

template <typename T> constexpr int kQueryParts = sizeof(T) == 4 ? 3 : std::is_same<T, _Float16>::value ? 2 : 1;
template <typename T> constexpr int kPowerParts = sizeof(T) == 4 ? 3 : 2;

struct Held { const void *k, *k_scales, *v, *v_scales; };
struct Results { void *out; float *part; float2 *part_stats; };

// How 32 keys of a cache come to a wavefront's lanes.  Keys: lane (g, c) takes chunks of rows c and 16 + c, the g-th of each four.  Values: chunks of
// all rows one after the other.
template <int D, int BITS> struct Layout {
    static constexpr int kRow = D * BITS / 8;
    static constexpr int kKeyBytes = kRow / 4, kKeyChunk = kKeyBytes < 16 ? kKeyBytes : 16, kKeyChunks = kKeyBytes / kKeyChunk;
    static constexpr int kKeyElements = kKeyChunk * 8 / BITS;
    static constexpr int kValueBytes = kRow / 2, kValueChunk = kValueBytes < 16 ? kValueBytes : 16, kValueChunks = kValueBytes / kValueChunk;
    static constexpr int kValueElements = kValueChunk * 8 / BITS, kPerRow = kRow / kValueChunk;
    // first of the elements 8 n .. 8 n + 7 of lane group g
    static __device__ __forceinline__ int element(int n, int g) { return (8 * n / kKeyElements * 4 + g) * kKeyElements + 8 * n % kKeyElements; }
};

template <int BYTES> __device__ __forceinline__ void load_words(const uint8_t *p, uint32_t *w) {
    if constexpr (BYTES == 16) {
        const u32x4 x = *reinterpret_cast<const u32x4 *>(p);
        w[0] = x[0]; w[1] = x[1]; w[2] = x[2]; w[3] = x[3];
    } else if constexpr (BYTES == 8) {
        const uint2 x = *reinterpret_cast<const uint2 *>(p);
        w[0] = x.x; w[1] = x.y;
    } else {
        w[0] = *reinterpret_cast<const uint32_t *>(p);
    }
}

template <int D, int BITS> struct Step {
    typedef Layout<D, BITS> Y;
    int key0;
    uint32_t kw[2][Y::kKeyBytes / 4], vw[Y::kValueBytes / 4];
    unsigned ks[2][Y::kKeyChunks], vs[Y::kValueChunks];

    // Rows behind the last key read it again: what a padded cache holds there is never touched.  Whole steps are addressed from one place for all lanes.
    __device__ __forceinline__ void fetch(const Rows<D, BITS> &k, const Rows<D, BITS> &v, int first, int k_len, int lane) {
        key0 = first;
        const int64_t at = first;
        if (first + kUnit <= k_len) fetch_rows(Rows<D, BITS>{k, at}, Rows<D, BITS>{v, at}, lane, [](int r) { return r; });
        else fetch_rows(Rows<D, BITS>{k, at}, Rows<D, BITS>{v, at}, lane, [&](int r) { return min(r, k_len - 1 - first); });
    }
    template <typename F> __device__ __forceinline__ void fetch_rows(const Rows<D, BITS> k, const Rows<D, BITS> v, int lane, F row_of) {
        const int g = lane >> 4, c = lane & 15;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            const int row = row_of(16 * kt + c);
#pragma unroll
            for (int j = 0; j < Y::kKeyChunks; ++j) {
                load_words<Y::kKeyChunk>(k.codes + (row * Y::kRow + (4 * j + g) * Y::kKeyChunk), kw[kt] + j * Y::kKeyChunk / 4);
                ks[kt][j] = k.scales[row * (D / kGroup) + (4 * j + g) * Y::kKeyElements / kGroup];
            }
        }
#pragma unroll
        for (int j = 0; j < Y::kValueChunks; ++j) {
            const int at = j * 64 + lane, col = at % Y::kPerRow, row = row_of(at / Y::kPerRow);
            load_words<Y::kValueChunk>(v.codes + (row * Y::kRow + col * Y::kValueChunk), vw + j * Y::kValueChunk / 4);
            vs[j] = v.scales[row * (D / kGroup) + col * Y::kValueElements / kGroup];
        }
    }
    // The largest scale of the lane's values: 255 where some are no numbers.
    __device__ __forceinline__ unsigned most() const {
        unsigned most = 0;
#pragma unroll
        for (int j = 0; j < Y::kValueChunks; ++j) most = max(most, vs[j]);
        return most;
    }
    // For all lanes, where any has such values: these become 0, and each key's mark has a bit for each 32 of them.
    __device__ __forceinline__ void clear(uint8_t *marks, int lane) {
#pragma unroll
        for (int j = 0; j < Y::kValueChunks; ++j) {
            unsigned mark = vs[j] == 255 ? 1u << ((j * 64 + lane) % Y::kPerRow * Y::kValueElements / kGroup) : 0u;
            if (mark)
#pragma unroll
                for (int i = 0; i < Y::kValueChunk / 4; ++i) vw[j * Y::kValueChunk / 4 + i] = 0;
            vs[j] = mark ? 0 : vs[j];
            // a row's chunks lie in neighbouring lanes
#pragma unroll
            for (int d = 1; d < Y::kPerRow; d <<= 1) mark |= __shfl_xor(mark, d);
            if (lane % Y::kPerRow == 0) marks[(j * 64 + lane) / Y::kPerRow] = (uint8_t)mark;
        }
    }
    __device__ __forceinline__ bf16x8 keys(int kt, int n) const {
        constexpr int W = BITS / 4;
        return values<BITS>(kw[kt] + n * W, scale_of(ks[kt][8 * n / Y::kKeyElements]));
    }
    __device__ __forceinline__ void store_values(__bf16 *stage, int lane) const {
        constexpr int W = BITS / 4, S = D + kPad;
#pragma unroll
        for (int j = 0; j < Y::kValueChunks; ++j) {
            const int at = j * 64 + lane;
            __bf16 *to = stage + at / Y::kPerRow * S + at % Y::kPerRow * Y::kValueElements;
#pragma unroll
            for (int n = 0; n < Y::kValueElements / 8; ++n)
                *reinterpret_cast<bf16x8 *>(to + 8 * n) = values<BITS>(vw + j * Y::kValueChunk / 4 + n * W, scale_of(vs[j]));
        }
    }
};

// Eight elements of a query as a sum of bfloat16.  Cut, not rounded: a part never leaves the range.
template <typename T> __device__ __forceinline__ void parts_of(const T *src, bf16x8 *part, int stride) {
    const V8<T> x = load8(src);
    if constexpr (std::is_same<T, __bf16>::value) {
        part[0] = x;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float f = (float)x[i];
#pragma unroll
            for (int j = 0; j < kQueryParts<T>; ++j) {
                const float high = __uint_as_float(__float_as_uint(f) & 0xffff0000u);
                part[j * stride][i] = (__bf16)high;
                f = fabsf(f) < __builtin_inff() ? f - high : 0.f;
            }
        }
    }
}

// The queries of a lane's column as operands: D / 32 times eight elements, the first of the n-th from element_of(n) on.
template <typename T, int D, typename F>
__device__ __forceinline__ void load_queries(const Problem &p, int b, int t, int head, bool there, bf16x8 (&q)[kQueryParts<T>][D / 32], F element_of) {
    const T *src = static_cast<const T *>(p.q) + b * p.qs.batch + (int64_t)t * p.qs.row + head * p.qs.head;
#pragma unroll
    for (int n = 0; n < D / 32; ++n) {
        if (there && p.scale2 != 0.f) {
            parts_of<T>(src + element_of(n), &q[0][n], D / 32);
        } else {
#pragma unroll
            for (int j = 0; j < kQueryParts<T>; ++j) q[j][n] = zero8<__bf16>();
        }
        if (p.scale2 < 0.f)
#pragma unroll
            for (int j = 0; j < kQueryParts<T>; ++j) q[j][n] = -q[j][n];
    }
}
// Scores are compared before they are scaled: a negative scale turns the queries' signs instead, and one of 0 takes the queries away.
__device__ __forceinline__ float factor_of(const Problem &p) { return p.scale2 == 0.f ? 1.f : fabsf(p.scale2); }

// Last key that a lane's row may see; columns that no row of the result belongs to see everything, so that they do not keep a tile from skipping its masks.
__device__ __forceinline__ int limit_of(const Problem &p, bool used, int t, int q_len, int k_len) {
    if (!used || t >= p.queries) return k_len - 1;
    return t >= q_len ? -1 : p.causal ? min(k_len - q_len + t, k_len - 1) : k_len - 1;
}

// One row's softmax: powers are relative to `m`, which follows the largest score when that has moved by more than 2^8; their sum is any of `sum` (a product with ones
// makes it, of the parts that weigh the values); `lost` are the parts of 32 elements that are NaN.
// Sums are divided at the end.  Of 2^30 keys, the most there are, with powers of up to 2^8 and elements of up to 448 x 2^80 they stay below 2^127; caches hold elements of
// up to 2^128.  Where a step has a larger scale than 2^80 the reference goes to kLift above its largest score, which keeps its powers below 2^-kLift.  Powers are
// then rounded to 2^-19 of themselves by their exponents, and lost below 2^-86, which is why this is not done for all.
constexpr unsigned kLargeScale = 127 + 80;
constexpr float kLift = 40.f;
template <int D> struct Row {
    float m;
    unsigned lost;
    f32x4 sum, o[D / 16];
    __device__ __forceinline__ void clear() {
        m = -__builtin_inff(); lost = 0;
        sum = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    // Scores s of keys key0 + 16 kt + 4 g + i, of which the row sees those up to `last`: the others become -inf.
    static __device__ __forceinline__ void mask(f32x4 (&s)[2], int key0, int g, int last) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[kt][i] = key0 + 16 * kt + 4 * g + i <= last ? s[kt][i] : -__builtin_inff();
    }
    // A row whose own largest score has not moved is multiplied by 1, whoever stands beside it.
    __device__ __forceinline__ void follow(float top, bool large) {
        const float at = large ? top + kLift : top;
        const bool moved = large ? at > m : top > m + 8.f;
        const float to = moved ? at : m, shrink = moved ? __builtin_amdgcn_exp2f(m - to) : 1.f;
        sum *= shrink;
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) o[dt] *= shrink;
        m = to;
    }
    // The scores' powers, in parts.
    template <int NP> __device__ __forceinline__ void powers(const f32x4 (&s)[2], float factor, bf16x8 (&part)[NP]) {
        const float ref = m == -__builtin_inff() ? 0.f : m;           // nothing above -inf so far: every power is 0
        f32x4 z[2];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int i = 0; i < 4; ++i) z[kt][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][i], factor, -ref));
        bf16x8 ones;
#pragma unroll
        for (int i = 0; i < 8; ++i) ones[i] = (__bf16)1.f;
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            part[j] = pack<__bf16>(z[0], z[1]);
            sum = mma(ones, part[j], sum);
            if (j + 1 < NP)
#pragma unroll
                for (int i = 0; i < 4; ++i) { z[0][i] -= (float)part[j][i]; z[1][i] -= (float)part[j][4 + i]; }
        }
    }
    // Marks of 32 keys, a byte each.
    __device__ __forceinline__ void mark(const uint8_t *marks, int key0, int g, int last) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int key = 16 * (i >> 2) + 4 * g + (i & 3);
            lost |= key0 + key <= last ? marks[key] : 0u;
        }
    }
    __device__ __forceinline__ void lose() {
        if (!__any(lost != 0)) return;
        unsigned bad = lost | __shfl_xor(lost, 16);
        bad |= __shfl_xor(bad, 32);
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt)
            if (bad >> (dt / 2) & 1) o[dt] = f32x4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
    }
};

// Four consecutive elements of a result.
template <typename T> __device__ __forceinline__ void store_result(T *out, int64_t at, f32x4 v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = within<T>(v[i]);
    store_row<T>(out, nullptr, at, v);
}

constexpr int kListed = 1024;          // blocks listed at a time
struct NoList {};

// Wavefronts of a SIMD that registers are left for: 128, 168 or 256 each; as many as spill nothing.  One token over 32 x 32,768 keys of 8 x 128 (us): bfloat16 / 4 bits (four) 199, float16 / 4 (three) 201,
// bfloat16 / 8 (three) 381, float16 / 8 with two 385, with three and 24 bytes in scratch 380, over 32,768 keys alone 19.5 and 20.0, 4 tokens over 8 x 4,096 20.1 and 20.9; float32 (two) 227 and 386.
template <typename T, int D, int BITS, int RT, bool LISTED>
constexpr int kResident = RT > 1 ? 2
    : D < 128 ? 4 - (sizeof(T) == 4 && BITS == 8 && LISTED)
    : sizeof(T) == 4 || (std::is_same<T, _Float16>::value && BITS == 8) ? 2
    : (BITS == 4 && std::is_same<T, __bf16>::value ? 4 : 3) - LISTED;
// Most tiles of 16 rows that a workgroup takes.
template <typename T, int D> constexpr int kMostTiles = sizeof(T) == 4 && D == 128 ? 1 : 2;

// Floats between rows, and between wavefronts, of the joining buffer: neighbours lie on other banks.
template <int D> constexpr int kMergeRow = D + 4;
template <int D> constexpr int kMergeWave = 16 * kMergeRow<D> + 4;

template <int D> constexpr size_t stage_bytes() {
    const size_t values = (size_t)kWaves * kUnit * (D + kPad) * sizeof(__bf16), merge = (size_t)kWaves * kMergeWave<D> * sizeof(float);
    return values > merge ? values : merge;
}

template <typename T, int D, int BITS, int RT, bool LISTED>
__global__ __launch_bounds__(kThreads, (kResident<T, D, BITS, RT, LISTED>)) void attention_kernel(const Problem p, const Held held, const Results r, int n_groups, int splits) {
    constexpr int DC = D / 32, DT = D / 16, NQ = kQueryParts<T>, NP = kPowerParts<T>;
    typedef List<RT, kListed> Listing;
    __shared__ typename std::conditional<LISTED, Listing, NoList>::type list;
    __shared__ float2 stats[kWaves][16], joined[16];
    __shared__ uint8_t marks[kWaves][kUnit];
    __shared__ __align__(16) unsigned char dynamic[stage_bytes<D>()];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, c = lane & 15;
    const int unit = xcd_contiguous_block(), pair = unit / (n_groups * splits), rest = unit - pair * n_groups * splits;
    const int group = rest / splits, split = rest - group * splits;
    const int b = pair / p.kv_heads, h = pair - b * p.kv_heads;
    const int k_len = key_count(p, b), q_len = query_count(p, b), offset = k_len - q_len;
    const int tpt = tile_tokens(p.group), t0 = group * RT * tpt;
    const int tc = c / p.group, mine = c - tc * p.group, head = h * p.group + mine;        // this lane's token within a tile, and its head
    const bool used = tc < tpt;

    __bf16 *stage = reinterpret_cast<__bf16 *>(dynamic) + wave * kUnit * (D + kPad);
    const Rows<D, BITS> keys(held.k, held.k_scales, pair, p.keys), vals(held.v, held.v_scales, pair, p.keys);
    const float factor = factor_of(p);
    bf16x8 qf[RT][NQ][DC];
    int limit[RT];
    Row<D> row[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int t = t0 + rt * tpt + tc;
        limit[rt] = limit_of(p, used, t, q_len, k_len);
        row[rt].clear();
        load_queries<T, D>(p, b, t, head, used && t < q_len, qf[rt], [&](int n) { return Layout<D, BITS>::element(n, g); });
    }
    // rows behind the queries see nothing, and no keys are walked for them (64 sequences padded to 64 tokens, 4,096 keys of 8 x 128 in 4 bits: with 1 token each 254 us, walking 441; with none 34 and 450)
    const int last_key = t0 >= q_len ? -1 : p.causal ? min(k_len - 1, offset + min(t0 + RT * tpt, q_len) - 1) : k_len - 1;
    const int sub_shift = LISTED ? p.block_shift - 5 : 0, stride = kWaves * splits;

    auto window = [&](int first, int units) {
        auto first_key = [&](int u) {
            if constexpr (LISTED) return __builtin_amdgcn_readfirstlane(((first + list.id[u >> sub_shift]) << p.block_shift) + ((u & ((1 << sub_shift) - 1)) << 5));
            else return u << 5;
        };
        // the next unit, from u on, that holds a key anyone may see
        auto find = [&](int u) {
            if constexpr (LISTED)
                while (u < units && first_key(u) > last_key) u += stride;
            return u;
        };
        Step<D, BITS> step;
        unsigned who[RT];              // tokens of each tile that selected these keys
        auto fetch = [&](int u) {
            step.fetch(keys, vals, first_key(u), k_len, lane);
            if constexpr (LISTED)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) who[rt] = (unsigned)(list.bits[u >> sub_shift][0] >> (16 * rt)) & 0xffffu;
        };
        int u = find(wave + kWaves * split);
        if (u < units) fetch(u);
        while (u < units) {
            const int key0 = step.key0;
            int last[RT];              // keys that the lane's row sees: key0 + 16 kt + 4 g + i <= last
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) last[rt] = !LISTED || !used || t0 + rt * tpt + tc >= p.queries || (who[rt] >> tc) & 1 ? limit[rt] : -1;
            wave_lds_sync();
            bool odd = false, large = false;       // of all lanes
            if (__any(step.most() > kLargeScale)) {
                odd = __any(step.most() == 255);
                if (odd) step.clear(marks[wave], lane);
                large = __any(step.most() > kLargeScale);
            }
            step.store_values(stage, lane);
            f32x4 s[RT][2];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) s[rt][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int n = 0; n < DC; ++n) {
                    const bf16x8 kf = step.keys(kt, n);
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                        for (int j = NQ; j-- > 0;) s[rt][kt] = mma(kf, qf[rt][j][n], s[rt][kt]);
                }
            }
            u = find(u + stride);
            if (u < units) fetch(u);
            wave_lds_sync();
            // each part of the softmax for all tiles, so that their chains run side by side
            bool edge = false, moved = false;
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) edge |= key0 + kUnit - 1 > last[rt];
            if (__any(edge))
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) Row<D>::mask(s[rt], key0, g, last[rt]);
            float top[RT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                top[rt] = largest_of_rows(largest(s[rt][0], s[rt][1])) * factor;
                moved |= top[rt] > row[rt].m + 8.f;
            }
            if (large || __any(moved))
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) row[rt].follow(top[rt], large);
            bf16x8 pf[RT][NP];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) row[rt].powers(s[rt], factor, pf[rt]);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const bf16x8 vf = transposed<__bf16, D>(stage, dt * 16, lane);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int j = 0; j < NP; ++j) row[rt].o[dt] = mma(vf, pf[rt][j], row[rt].o[dt]);
            }
            if (odd)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) row[rt].mark(marks[wave], key0, g, last[rt]);
        }
    };
    if constexpr (LISTED) {
        for (int first = 0; first < p.blocks; first += kListed)
            window(first, build_list(list, p, b, h, t0, q_len, k_len, first, min(kListed, p.blocks - first)) << sub_shift);
    } else {
        window(0, (last_key + kUnit) / kUnit);
    }

    // the wavefronts' sums, joined: the threads of a workgroup share the columns out, and where there are more of them the wavefronts too
    constexpr int ITEMS = 16 * D / 4, SHARE = kThreads > ITEMS ? kThreads / ITEMS : 1, STEP = kThreads / SHARE;
    float *merge = reinterpret_cast<float *>(dynamic);
    const int64_t all_rows = (int64_t)p.batch * p.queries * p.heads;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        row[rt].lose();
        if (g == 0) stats[wave][c] = make_float2(row[rt].m, row[rt].sum[0]);
        __syncthreads();               // the values' staging, or the joining buffer of the tile before, has been read
        float top = -__builtin_inff(), total = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) top = fmaxf(top, stats[w][c].x);
        const float ref = top == -__builtin_inff() ? 0.f : top;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) total += stats[w][c].y * __builtin_amdgcn_exp2f(stats[w][c].x - ref);
        const float share = __builtin_amdgcn_exp2f(row[rt].m - ref);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4 *>(merge + wave * kMergeWave<D> + c * kMergeRow<D> + 16 * dt + 4 * g) = row[rt].o[dt] * share;
        if (wave == 0 && g == 0) joined[c] = make_float2(top, total);
        __syncthreads();
#pragma unroll
        for (int item = tid / SHARE; item < ITEMS; item += STEP) {
            const int r16 = item / (D / 4), col = item % (D / 4) * 4, at_token = r16 / p.group, t = t0 + rt * tpt + at_token;
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = tid % SHARE; w < kWaves; w += SHARE) v += *reinterpret_cast<const f32x4 *>(merge + w * kMergeWave<D> + r16 * kMergeRow<D> + col);
            if constexpr (SHARE > 1)
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] += dpp_move<0xB1>(v[i]);        // two threads (heads of 32)
            if (tid % SHARE || at_token >= tpt || t >= p.queries) continue;
            const int64_t at = ((int64_t)b * p.queries + t) * p.heads + h * p.group + (r16 - at_token * p.group);
            const float2 st = joined[r16];
            if (splits == 1) {
                store_result<T>(static_cast<T *>(r.out), at * D + col, v * (st.y == 0.f ? 0.f : 1.f / st.y));
            } else {
                *reinterpret_cast<f32x4 *>(r.part + (split * all_rows + at) * D + col) = v;
                if (col == 0) r.part_stats[split * all_rows + at] = st;
            }
        }
    }
}

// Joins the shares of one row: the threads of a workgroup take four columns of every so many of them.
constexpr int kMostSplits = 256;
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void join_shares_kernel(const float *part, const float2 *part_stats, T *out, int64_t rows, int splits) {
    constexpr int C = D / 4, SUBS = kThreads / C;
    __shared__ float weight[kMostSplits];
    __shared__ f32x4 sums[SUBS][C];
    const int tid = threadIdx.x, lane = tid & 63, col = tid % C, sub = tid / C;
    const int64_t row = blockIdx.x;
    float top = -__builtin_inff(), total = 0.f;
    for (int s = lane; s < splits; s += 64) top = fmaxf(top, part_stats[s * rows + row].x);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
    const float ref = top == -__builtin_inff() ? 0.f : top;
    for (int s = lane; s < splits; s += 64) {
        const float2 st = part_stats[s * rows + row];
        const float w = __builtin_amdgcn_exp2f(st.x - ref);
        total += st.y * w;
        if (tid < 64) weight[s] = w;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) total += __shfl_xor(total, d);
    __syncthreads();
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = sub; s < splits; s += SUBS) v += *reinterpret_cast<const f32x4 *>(part + (s * rows + row) * D + col * 4) * weight[s];
    sums[sub][col] = v;
    __syncthreads();
    if (sub) return;
#pragma unroll
    for (int i = 1; i < SUBS; ++i) v += sums[i][col];
    store_result<T>(out, row * D + col * 4, v * (total == 0.f ? 0.f : 1.f / total));
}

// How a call's work is cut: where there are too few workgroups for the card, several share a row's keys out.  512 workgroups (two a CU) as long as each
// has eight steps of 32 keys for every tile, 256 as long as each wavefront has one; rows of up to 512 keys stay whole, for joining takes a launch of 3.5 us.
// Kernel and joining (us), shares as the rule has them / half / twice as many: 1 sequence of 8 key heads x 128, 4 bits, 32,768 keys (64 shares) 13.6 / 15.0 / 15.5, 8,192 keys (32) 8.5 / 10.4 /
// 9.1; 8 sequences of 4,096 (8) 13.1 / 14.6 / 13.8; 32 of 32,768 (2) 198 / 270 / 207; 1 of 2,048 x 8 heads x 64, 8 bits (16) 7.1 / 7.9 / 7.3; 3 tokens
// of 8 sequences, 16 blocks of 64 each (8) 11.0 / 12.7 / 12.0; 512 keys (1) 6.9, in four shares 7.1; 8 tokens over 16,384 keys (32) 15.4 / 18.9 / 18.6, 64 (8) 43 / 48 / 48.
// Workgroups take two tiles of rows where there are as many, which then share the work on the keys (64 tokens over 16,384 keys of 8 x 128, 8 bits: 43 us, with one tile 55); not with
// lists, whose unions grow.
struct Shape { int tiles, n_groups, splits; };
Shape shape_of(const Problem &p, int most_tiles) {
    const int tpt = tile_tokens(p.group);
    const int tiles = !p.topk && p.queries > tpt ? most_tiles : 1, tokens = tiles * tpt;
    Shape s{tiles, (int)(((int64_t)p.queries + tokens - 1) / tokens), 1};
    const int64_t groups = std::max<int64_t>((int64_t)p.batch * p.kv_heads * s.n_groups, 1);
    int64_t units = ((int64_t)p.keys + kUnit - 1) / kUnit;
    if (p.topk) units = std::min<int64_t>(units, ((int64_t)p.topk * std::min(tokens, p.queries)) << (p.block_shift - 5));
    if (units > 4 * kWaves)
        s.splits = (int)std::max<int64_t>(1, std::max(std::min({512 / groups, units / (2 * kWaves * s.tiles), (int64_t)kMostSplits}),
                                                      std::min({256 / groups, units / kWaves, (int64_t)kMostSplits})));
    return s;
}

size_t round_up(size_t n) { return (n + 255) & ~(size_t)255; }

template <typename T, int D, int BITS>
int launch(const Problem &p, const fg_cache_attention_args *a, void *workspace, size_t bytes, size_t *need, hipStream_t stream) {
    constexpr int MOST = kMostTiles<T, D>;
    const Shape s = shape_of(p, MOST);
    const size_t rows = (size_t)p.batch * p.queries * p.heads;
    const int64_t grid = (int64_t)p.batch * p.kv_heads * s.n_groups * s.splits;
    if (grid > kMostGroups) return fail(FG_ERR_SHAPE, "cache attention: %lld workgroups do not fit a launch", (long long)grid);
    const size_t sums = s.splits > 1 ? round_up(rows * s.splits * D * sizeof(float)) : 0, stats = s.splits > 1 ? round_up(rows * s.splits * sizeof(float2)) : 0;
    if (need) { *need = sums + stats; return FG_OK; }
    if (bytes < sums + stats || (sums && !workspace))
        return fail(FG_ERR_ARG, "cache attention: a workspace of %zu bytes, %zu needed (fg_cache_attention_workspace)", bytes, sums + stats);
    unsigned char *w = static_cast<unsigned char *>(workspace);
    const Results r{a->out, reinterpret_cast<float *>(w), reinterpret_cast<float2 *>(w + sums)};
    const Held held{a->cache.k, a->cache.k_scales, a->cache.v, a->cache.v_scales};
    const dim3 blocks((unsigned)grid), threads(kThreads);
    if (p.topk) attention_kernel<T, D, BITS, 1, true><<<blocks, threads, 0, stream>>>(p, held, r, s.n_groups, s.splits);
    else if (s.tiles == 1) attention_kernel<T, D, BITS, 1, false><<<blocks, threads, 0, stream>>>(p, held, r, s.n_groups, s.splits);
    else attention_kernel<T, D, BITS, MOST, false><<<blocks, threads, 0, stream>>>(p, held, r, s.n_groups, s.splits);
    FG_HIP_TRY(hipGetLastError());
    if (s.splits == 1) return FG_OK;
    join_shares_kernel<T, D><<<dim3((unsigned)rows), threads, 0, stream>>>(r.part, r.part_stats, static_cast<T *>(r.out), (int64_t)rows, s.splits);
    FG_HIP_TRY(hipGetLastError());
    return FG_OK;
}

template <typename T, int D> int launch_b(const Problem &p, const fg_cache_attention_args *a, void *workspace, size_t bytes, size_t *need, hipStream_t stream) {
    return a->cache.bits == 4 ? launch<T, D, 4>(p, a, workspace, bytes, need, stream) : launch<T, D, 8>(p, a, workspace, bytes, need, stream);
}

template <typename T> int launch_d(const Problem &p, const fg_cache_attention_args *a, void *workspace, size_t bytes, size_t *need, hipStream_t stream) {
    switch (a->cache.head_len) {
    case 32: return launch_b<T, 32>(p, a, workspace, bytes, need, stream);
    case 64: return launch_b<T, 64>(p, a, workspace, bytes, need, stream);
    default: return launch_b<T, 128>(p, a, workspace, bytes, need, stream);
    }
}

int launch_t(const Problem &p, const fg_cache_attention_args *a, void *workspace, size_t bytes, size_t *need, hipStream_t stream) {
    switch (a->type) {
    case FG_TYPE_F32: return launch_d<float>(p, a, workspace, bytes, need, stream);
    case FG_TYPE_F16: return launch_d<_Float16>(p, a, workspace, bytes, need, stream);
    default: return launch_d<__bf16>(p, a, workspace, bytes, need, stream);
    }
}

constexpr const char *kWhat = "cache attention";

int problem_of(const fg_cache_attention_args *a, Problem *p, bool sizes_only) {
    if (!a) return fail(FG_ERR_ARG, "cache attention: arguments are a null pointer");
    int rc;
    if (sizes_only) {
        fg_kv_cache c = a->cache;
        c.k = c.v = c.k_scales = c.v_scales = reinterpret_cast<void *>(16);
        rc = check(&c);
    } else {
        rc = check(&a->cache);
    }
    if (rc) return rc;
    const fg_kv_cache &c = a->cache;
    if (a->type != FG_TYPE_F32 && a->type != FG_TYPE_F16 && a->type != FG_TYPE_BF16) return fail(FG_ERR_ARG, "cache attention: unknown type %d", a->type);
    if (a->queries < 0 || a->heads < 1) return fail(FG_ERR_ARG, "cache attention: negative sizes, or no heads");
    if (a->heads % c.kv_heads || a->heads / c.kv_heads > 16)
        return fail(FG_ERR_SHAPE, "cache attention: %d heads over %d key heads: the former have to be 1 to 16 times the latter", a->heads, c.kv_heads);
    if (a->queries > (1 << 30)) return fail(FG_ERR_SHAPE, "cache attention: more than 2^30 queries");
    const bool listed = a->topk != 0;
    if (listed) {
        if (a->topk < 0) return fail(FG_ERR_ARG, "cache attention: %d blocks a query", a->topk);
        if (a->block != 32 && a->block != 64 && a->block != 128 && a->block != 256) return fail(FG_ERR_SHAPE, "cache attention: blocks of 32, 64, 128 or 256 keys, got %d", a->block);
        if ((int64_t)a->topk * 128 > INT32_MAX / c.kv_heads) return fail(FG_ERR_SHAPE, "cache attention: too long a list");
    }
    *p = Problem{};
    if ((rc = strides_of("q", a->q, a->q_strides, a->type == FG_TYPE_F32 ? 4 : 2, &p->qs, kWhat)) || (rc = aligned("out", a->out, 16, kWhat)) ||
        (rc = aligned("blocks", a->blocks, 4, kWhat)) || (rc = aligned("lengths", a->lengths, 4, kWhat)) ||
        (rc = aligned("q_lengths", a->q_lengths, 4, kWhat))) return rc;
    p->batch = c.batch; p->queries = a->queries; p->keys = c.keys; p->heads = a->heads; p->kv_heads = c.kv_heads; p->group = a->heads / c.kv_heads;
    p->causal = a->causal != 0; p->scale = a->scale; p->scale2 = a->scale * kLog2e;
    p->q = a->q; p->lengths = a->lengths; p->q_lengths = a->q_lengths;
    if (listed) {
        p->block_shift = a->block == 32 ? 5 : a->block == 64 ? 6 : a->block == 128 ? 7 : 8;
        p->blocks = (c.keys + a->block - 1) / a->block;
        p->topk = a->topk;
        p->list = a->blocks;
    }
    return FG_OK;
}

}  // namespace
}  // namespace cache
}  // namespace fg

extern "C" int64_t fg_cache_attention_workspace(const fg_cache_attention_args *args) {
    fg::block::Problem p;
    if (int rc = fg::cache::problem_of(args, &p, true)) return rc;
    size_t need = 0;
    const int rc = fg::cache::launch_t(p, args, nullptr, 0, &need, nullptr);
    return rc ? rc : (int64_t)need;
}

extern "C" int fg_cache_attention(const fg_cache_attention_args *args, void *workspace, size_t workspace_bytes, void *stream) {
    fg::block::Problem p;
    if (int rc = fg::cache::problem_of(args, &p, false)) return rc;
    if ((int64_t)p.batch * p.queries == 0) return FG_OK;
    if (!p.q || !args->out || (p.topk && !p.list)) return fg::fail(FG_ERR_ARG, "cache attention: null pointer");
    if (int rc = fg::block::aligned("the workspace", workspace, 16, "cache attention")) return rc;
    return fg::cache::launch_t(p, args, workspace, workspace_bytes, nullptr, static_cast<hipStream_t>(stream));
}
