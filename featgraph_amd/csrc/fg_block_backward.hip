// Gradients of attention over selected blocks of keys.  With p_ij = 2^(z_ij - m_i - log2 l_i) the forward pass's softmax:
//   dP_ij = <dO_i, V_j>,  dS_ij = p_ij (dP_ij - delta_i),  delta_i = <dO_i, O_i>
//   dQ_i = scale sum_j dS_ij K_j,  dK_j = scale sum_i dS_ij Q_i,  dV_j = sum_i p_ij dO_i,  dbias[n, h] = sum of dS_ij in bucket n
//
// Two sweeps form the scores again.  queries_kernel goes by query like the forward pass (its list of blocks, dQ and dbias).  keys_kernel goes by block:
// the lists are turned round -- for every block the tokens that selected it, in order -- and a workgroup takes a block, or a piece of a long
// list, with its keys in registers, and gathers the rows of its tokens' heads.  Nothing is added by atomics: sums over pieces,
// wavefronts and tiles are joined in a fixed order, so that a step gives the same bits every time.
//
// What bounds them (2 x 4,096 tokens, 16 / 4 heads of 128 in bfloat16, 16 blocks of 64): queries_many_kernel 278 us, as the forward pass,
// with two products more; keys_kernel 369 us: one wavefront per SIMD (sums of 32 keys, their operands and the rows under way take 398
// registers), so that every wait shows, and 70 us of beginnings and ends of 1,100 pieces; the lists 24 us in four launches, the sums of
// pieces 14 (5 TB/s).  With heads of 64 two wavefronts fit (8,192 tokens, 16 / 1 heads, 8 blocks of 128 in float16: 152 and 206 us, 7 of them
// for the scale of dS).
#include <algorithm>
#include <type_traits>

#include "fg_block.h"

namespace fg {
namespace block {

namespace {

constexpr int kMergeStride = 36;       // floats between rows of the joining buffer (32 and 4 of padding)
constexpr int kWindow = 1024;          // blocks looked at together

struct Piece { int32_t block, start, len, slot; };     // block: of all sequences and key heads; slot: where its sums go, -1: they are all

// ---- lists by block ---------------------------------------------------------------------------------------

// bits[pair][chunk][block]: which of the chunk's 64 tokens selected the block.
__global__ __launch_bounds__(kThreads) void mark_kernel(const Problem p, unsigned long long *bits, int chunks) {
    __shared__ unsigned long long mask[kWindow];
    const int chunk = blockIdx.x % chunks, pair = blockIdx.x / chunks, b = pair / p.kv_heads, h = pair - b * p.kv_heads, t0 = chunk * 64;
    const int k_len = key_count(p, b), q_len = query_count(p, b), offset = k_len - q_len, there = min(64, q_len - t0);
    const int64_t row = (int64_t)p.kv_heads * p.topk;
    const int32_t *src = p.list + ((int64_t)b * p.queries + t0) * row + (int64_t)h * p.topk;
    unsigned long long *dst = bits + ((int64_t)pair * chunks + chunk) * p.blocks;
    for (int first = 0; first < p.blocks; first += kWindow) {
        const int width = min(kWindow, p.blocks - first);
        __syncthreads();
        for (int i = threadIdx.x; i < width; i += kThreads) mask[i] = 0;
        __syncthreads();
        for (int e = threadIdx.x; e < there * p.topk; e += kThreads) {
            const int t = e / p.topk, blk = src[t * row + (e - t * p.topk)], at = blk - first;
            if (at < 0 || at >= width) continue;
            const int key = blk << p.block_shift;
            if (key < k_len && (!p.causal || key <= offset + t0 + t)) atomicOr(&mask[at], 1ull << t);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < width; i += kThreads) dst[first + i] = mask[i];
    }
}

// count[m] of block m = pair * blocks + block: one wavefront each.
__global__ __launch_bounds__(kThreads) void count_kernel(const unsigned long long *bits, int32_t *count, int all, int blocks, int chunks) {
    const int m = blockIdx.x * kWaves + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (m >= all) return;
    const int pair = m / blocks;
    const unsigned long long *src = bits + (int64_t)pair * chunks * blocks + (m - pair * blocks);
    int n = 0;
    for (int c = lane; c < chunks; c += 64) n += __popcll(src[(int64_t)c * blocks]);
#pragma unroll
    for (int d = 32; d; d >>= 1) n += __shfl_xor(n, d);
    if (lane == 0) count[m] = n;
}

// Where each block's tokens, whole pieces and partial sums begin; totals[0]: all whole pieces.  One workgroup.
constexpr int kScan = 1024;
__global__ __launch_bounds__(kScan) void scan_kernel(const int32_t *count, int32_t *offset, int32_t *piece0, int32_t *slot0, int32_t *totals, int all, int piece) {
    __shared__ int sums[3][kScan / 64];
    int base[3] = {0, 0, 0};
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int m0 = 0; m0 < all; m0 += kScan) {
        const int m = m0 + tid, n = m < all ? count[m] : 0, k = (n + piece - 1) / piece;
        const int own[3] = {n, n / piece, k > 1 ? k : 0};
        int upto[3] = {own[0], own[1], own[2]};
#pragma unroll
        for (int x = 0; x < 3; ++x) {
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int o = __shfl_up(upto[x], d);
                if (lane >= d) upto[x] += o;
            }
            if (lane == 63) sums[x][wave] = upto[x];
        }
        __syncthreads();
        int total[3] = {0, 0, 0};
#pragma unroll
        for (int x = 0; x < 3; ++x) {
            for (int w = 0; w < kScan / 64; ++w) {
                if (w == wave) upto[x] += total[x];
                total[x] += sums[x][w];
            }
        }
        if (m < all) {
            offset[m] = base[0] + upto[0] - own[0];
            piece0[m] = base[1] + upto[1] - own[1];
            slot0[m] = base[2] + upto[2] - own[2];
        }
#pragma unroll
        for (int x = 0; x < 3; ++x) base[x] += total[x];
        __syncthreads();
    }
    if (tid == 0) totals[0] = base[1];
}

// Short sequences, whose lists are never cut: a place for every query in every block's list, which one wavefront per block finds by looking
// through the selections themselves.
__global__ __launch_bounds__(kThreads) void short_lists_kernel(const Problem p, int32_t *count, int32_t *list, int all) {
    const int m = blockIdx.x * kWaves + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (m >= all) return;
    const int pair = m / p.blocks, blk = m - pair * p.blocks, b = pair / p.kv_heads, h = pair - b * p.kv_heads, key = blk << p.block_shift;
    const int k_len = key_count(p, b), q_len = query_count(p, b), offset = k_len - q_len;
    const int64_t row = (int64_t)p.kv_heads * p.topk;
    const int32_t *src = p.list + (int64_t)b * p.queries * row + (int64_t)h * p.topk;
    int32_t *dst = list + (int64_t)m * p.queries;
    int n = 0;
    // causal queries before the block do not see it
    for (int t0 = p.causal ? max(key - offset, 0) & ~63 : 0; t0 < q_len; t0 += 64) {
        const int t = t0 + lane;
        bool named = false;
        for (int j = 0; j < p.topk; ++j) named |= src[min(t, q_len - 1) * row + j] == blk;
        const unsigned long long all_named = __ballot(named && t < q_len && key < k_len && (!p.causal || key <= offset + t));
        if ((all_named >> lane) & 1) dst[n + __popcll(all_named & ((1ull << lane) - 1))] = t;
        n += __popcll(all_named);
    }
    if (lane == 0) count[m] = n;
}

// The tokens of every block in ascending order, and its pieces: one wavefront per block.  Whole pieces of all blocks come first, then what is
// left of every block's list (len 0: nothing chose the block; -1: nothing is left), so that the short ones fill the card's last round.
__global__ __launch_bounds__(kThreads) void fill_kernel(const unsigned long long *bits, const int32_t *count, const int32_t *offset, const int32_t *piece0,
                                                        const int32_t *slot0, const int32_t *totals, int32_t *list, Piece *pieces, int all, int blocks, int chunks, int piece) {
    const int m = blockIdx.x * kWaves + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (m >= all) return;
    const int pair = m / blocks, n = count[m], whole = n / piece, left = n - whole * piece, k = whole + (left > 0), at0 = offset[m];
    for (int i = lane; i < whole; i += 64) pieces[piece0[m] + i] = Piece{m, at0 + i * piece, piece, k > 1 ? slot0[m] + i : -1};
    if (lane == 0) pieces[totals[0] + m] = Piece{m, at0 + whole * piece, left || !whole ? left : -1, k > 1 ? slot0[m] + whole : -1};
    const unsigned long long *src = bits + (int64_t)pair * chunks * blocks + (m - pair * blocks);
    int base = at0;
    for (int c0 = 0; c0 < chunks; c0 += 64) {
        unsigned long long w = c0 + lane < chunks ? src[(int64_t)(c0 + lane) * blocks] : 0;
        const int own = __popcll(w);
        int upto = own;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(upto, d);
            if (lane >= d) upto += o;
        }
        int at = base + upto - own;
        for (; w; w &= w - 1) list[at++] = (c0 + lane) * 64 + __builtin_ctzll(w);
        base += __shfl(upto, 63);
    }
}

// ---- by query: dQ, dbias and delta ------------------------------------------------------------------------

struct Step { const void *dout, *out, *rest; Strides ds; const float2 *lse; float *delta; float2 *largest; void *dq; float *bias_sums; };

// float16 holds numbers from 6e-5 (in full) to 65504, and dS has the gradients' range: loss scaling moves it, but between rows and heads it
// remains wide.  So dS enters its products times a power of two and the sums are taken back in 32 bits.  By query every row has its own, 2^up:
// 2^kRoom over |dO_i| |O_i|, where dS = p <dO_i, V_j - O_i> is of the size of p 2^kRoom, or of some times that.  A row whose values nearly cancel
// one another makes it infinite: it is computed again, as tiles with infinities are, with 2^kSafeRoom over |dO_i|, which nothing
// finite can exceed: |dS| <= |dO_i| max |V| / 2, and 128 elements of 65504 are |V| < 2^19.5.  By key see keys_kernel.
template <typename T> constexpr bool kNarrow = std::is_same<T, _Float16>::value;
constexpr int kRoom = 8, kSafeRoom = -4;

// A lane's row of a tile: dO and Q as operands, and delta.
template <typename T, int D> struct Row16 {
    V8<T> q[D / 32], d[D / 32];
    // p is 2^(z - lse) weight, and dS is 2^(z - lse) (dP weight - less): the row's sum is a factor of the second one, in one operation, and never
    // added to the reference, which from 2^24 on would take it away
    float lse, weight, less, down;     // in float16 weight and less are 2^up times that, down is 2^-up
    float delta, more;
    float norm;                        // |dO|
    int up, safe_up;
    int limit;                         // last key that it may see; columns without a row see everything, nothing is written of them
    __device__ __forceinline__ void load(const Problem &p, const Step &w, int b, int t, int head, bool used, int q_len, int k_len, int offset, int g, bool write) {
        const bool there = used && t < q_len;
        limit = there ? (p.causal ? min(offset + t, k_len - 1) : k_len - 1) : used ? -1 : k_len - 1;
        const int64_t at = ((int64_t)b * p.queries + t) * p.heads + head;
        const T *qs = static_cast<const T *>(p.q) + b * p.qs.batch + (int64_t)t * p.qs.row + head * p.qs.head + 8 * g;
        const T *dos = static_cast<const T *>(w.dout) + b * w.ds.batch + (int64_t)t * w.ds.row + head * w.ds.head + 8 * g;
        const T *os = static_cast<const T *>(w.out) + at * D + 8 * g, *rs = static_cast<const T *>(w.rest) + at * D + 8 * g;
        float sum = 0.f, squares = 0.f, of_out = 0.f;
#pragma unroll
        for (int dc = 0; dc < D / 32; ++dc) {
            q[dc] = there ? load8(qs + dc * 32) : zero8<T>();
            d[dc] = there ? load8(dos + dc * 32) : zero8<T>();
            const V8<T> o = there ? load8(os + dc * 32) : zero8<T>();
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += (float)d[dc][i] * (float)o[i];
            if (kNarrow<T>)
#pragma unroll
                for (int i = 0; i < 8; ++i) { squares += (float)d[dc][i] * (float)d[dc][i]; of_out += (float)o[i] * (float)o[i]; }
            if (w.rest) {
                const V8<T> r = there ? load8(rs + dc * 32) : zero8<T>();
#pragma unroll
                for (int i = 0; i < 8; ++i) sum += (float)d[dc][i] * ((float)r[i] * (1.f / kRestScale<T>));
            }
        }
        delta = rows_sum(sum);
        const float2 ls = there ? w.lse[at] : make_float2(__builtin_inff(), 0.f);
        lse = ls.x;
        more = ls.y;
        if (there && write && g == 0) w.delta[at] = delta;
        norm = 0.f;
        up = safe_up = 0;
        if (kNarrow<T>) {
            squares = rows_sum(squares);
            of_out = rows_sum(of_out);
            const int size = (__builtin_amdgcn_frexp_expf(squares) + 1) >> 1;          // |dO| <= 2^size
            safe_up = kSafeRoom - size;
            up = of_out > 0.f ? kRoom - size - ((__builtin_amdgcn_frexp_expf(of_out) + 1) >> 1) : safe_up;
            norm = __builtin_sqrtf(squares);
        }
    }
    // The largest |dO| and |delta| of the tile that are finite, for the sweep by key (float16).
    __device__ __forceinline__ float2 largest() const {
        float2 v = make_float2(norm < __builtin_inff() ? norm : 0.f, fabsf(delta) < __builtin_inff() ? fabsf(delta) : 0.f);
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) { v.x = fmaxf(v.x, __shfl_xor(v.x, d)); v.y = fmaxf(v.y, __shfl_xor(v.y, d)); }
        return v;
    }
    __device__ __forceinline__ void weigh(bool safe) {
        const float by = kNarrow<T> ? (float)(safe ? safe_up : up) : 0.f;
        weight = __builtin_amdgcn_exp2f(by - more);
        less = delta * weight;
        down = __builtin_amdgcn_exp2f(-by);
    }
    // Whether a row of the wavefront is relative to a number, out of the bias, so large that adding the bias to the reference first would
    // leave other scores than the forward pass had.
    __device__ __forceinline__ bool far_off() const { return __any(fabsf(lse) > 4096.f && fabsf(lse) < __builtin_inff()); }
};

// The bias's gradient is summed in LDS, [wavefront][bucket][lane]: all rows of a lane have one head, and no two lanes a place.
__device__ __forceinline__ float *bias_place(const Problem &p, unsigned char *lds) {
    return reinterpret_cast<float *>(lds + ((buckets_bytes(p.n_buckets, p.low, p.high, p.group) + 15) & ~(size_t)15));
}
size_t bias_bytes(const Problem &p) {
    return p.n_buckets ? ((buckets_bytes(p.n_buckets, p.low, p.high, p.group) + 15) & ~(size_t)15) + (size_t)kWaves * p.n_buckets * 64 * sizeof(float) : 0;
}
// A workgroup's share of it, [workgroup of all sequences][head][bucket]; `more`: added to what it was.
__device__ __forceinline__ void write_bias(const Problem &p, const float *sums, float *out, int64_t workgroup, int h, bool more = false) {
    const int tpt = tile_tokens(p.group);
    __syncthreads();
    for (int e = threadIdx.x; e < p.n_buckets * p.group; e += kThreads) {
        const int x = e / p.n_buckets, n = e - x * p.n_buckets;
        float total = 0.f;
        for (int w = 0; w < kWaves; ++w)
            for (int t = 0; t < tpt; ++t)
                for (int q = 0; q < 4; ++q) total += sums[(w * p.n_buckets + n) * 64 + q * 16 + t * p.group + x];
        float *to = out + (workgroup * p.heads + h * p.group + x) * p.n_buckets + n;
        *to = more ? *to + total : total;
    }
}

// dS = 2^(z - lse) (dP weight - less) of one tile and 32 keys, into s[]: with MASK, keys behind `last` have none.  The bias's gradient goes to
// `sums`, times `down`.  far_off: the scores are formed as the forward pass does.
template <bool BIAS, bool MASK, bool NARROW>
__device__ __forceinline__ unsigned score_gradients(const Problem &p, const Buckets &buckets, float *sums, f32x4 *s, const f32x4 *dp, float lse, float weight, float less, float down, bool far_off,
                                                    int pos, int tpt, int tc, int mine, int key0, int last, int g, int lane) {
    const int near = BIAS ? buckets.at(pos - key0 - (kUnit - 1)) : 0, far = BIAS ? buckets.at(pos + tpt - 1 - key0) : 0;
    const float from = (BIAS && near == far ? buckets.value(near, mine) : 0.f) - (BIAS && far_off ? 0.f : lse);
    unsigned seen = MASK ? 0 : 0xff;
    float total = 0.f;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int key = key0 + 16 * kt + 4 * g + i;
            float z = s[kt][i] * p.scale2 + from;
            int bucket = 0;
            if (BIAS && near != far) {
                bucket = buckets.at(pos + tc - key);
                z += buckets.value(bucket, mine);
            }
            if (BIAS && far_off) z -= lse;
            float x = __builtin_amdgcn_exp2f(z) * (dp[kt][i] * weight - less);
            if (MASK) {
                x = key <= last ? x : 0.f;
                seen |= (unsigned)(key <= last) << (4 * kt + i);
            }
            s[kt][i] = x;
            if (BIAS) {
                if (near != far) sums[bucket * 64 + lane] += NARROW ? x * down : x;
                else total += x;
            }
        }
    if (BIAS && near == far) sums[near * 64 + lane] += NARROW ? total * down : total;
    return seen;
}

template <typename T, int D> constexpr size_t few_stage_bytes() {
    const size_t keys = (size_t)kWaves * kUnit * (D + kPad) * sizeof(T), merge = (size_t)kWaves * 16 * kMergeStride * sizeof(float);
    return keys > merge ? keys : merge;
}

// One tile of 16 rows, its list dealt out to the four wavefronts, as few_kernel does forward.
template <typename T, int D, bool CAREFUL>
__device__ __forceinline__ void few_rows(const Problem &p, const Step &w, List<1, kWindow> &list, unsigned char *dynamic, const Buckets &buckets, float *sums, int b, int h, int tile, float2 *largest) {
    constexpr int DC = D / 32, DT = D / 16, S = D + kPad;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, c = lane & 15;
    const int k_len = key_count(p, b), q_len = query_count(p, b), offset = k_len - q_len;
    const int tpt = tile_tokens(p.group), t0 = tile * tpt;
    const int tc = c / p.group, mine = c - tc * p.group, head = h * p.group + mine;
    const bool used = tc < tpt;
    T *stage = reinterpret_cast<T *>(dynamic) + wave * kUnit * S;
    Row16<T, D> row;
    row.load(p, w, b, t0 + tc, head, used, q_len, k_len, offset, g, wave == 0);
    const bool far_off = p.n_buckets && row.far_off();
    if (kNarrow<T> && largest && wave == 0) {
        const float2 v = row.largest();
        if (lane == 0) *largest = v;
    }
    const int last_key = p.causal ? min(k_len - 1, offset + min(t0 + tpt, q_len) - 1) : k_len - 1;
    const T *kbase = static_cast<const T *>(p.k) + b * p.ks.batch + h * p.ks.head + 8 * g;
    const T *vbase = static_cast<const T *>(p.v) + b * p.vs.batch + h * p.vs.head + 8 * g;
    const int sub_shift = p.block_shift - 5;

    f32x4 acc[DT];
    auto sweep = [&](auto careful) {
        for (int n = 0; n < p.n_buckets; ++n) sums[n * 64 + lane] = 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int first = 0; first < p.blocks; first += kWindow) {
            const int units = build_list(list, p, b, h, t0, q_len, k_len, first, min(kWindow, p.blocks - first)) << sub_shift;
            auto first_key = [&](int u) {
                return __builtin_amdgcn_readfirstlane(((first + list.id[u >> sub_shift]) << p.block_shift) + ((u & ((1 << sub_shift) - 1)) << 5));
            };
            auto find = [&](int u) {
                while (u < units && first_key(u) > last_key) u += kWaves;
                return u;
            };
            V8<T> kf[2][DC], vf[2][DC];
            int key0 = 0;
            unsigned who = 0;
            auto fetch = [&](int u) {
                key0 = first_key(u);
                who = (unsigned)list.bits[u >> sub_shift][0];
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) {
                    const int64_t key = min(key0 + kt * 16 + c, k_len - 1);
#pragma unroll
                    for (int dc = 0; dc < DC; ++dc) {
                        kf[kt][dc] = load8(kbase + key * p.ks.row + dc * 32);
                        vf[kt][dc] = load8(vbase + key * p.vs.row + dc * 32);
                    }
                }
            };
            int u = find(wave);
            if (u < units) fetch(u);
            while (u < units) {
                const int now = key0, last = !used || (who >> tc) & 1 ? row.limit : -1;
                wave_lds_sync();
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int dc = 0; dc < DC; ++dc) *reinterpret_cast<V8<T> *>(stage + (kt * 16 + c) * S + dc * 32 + 8 * g) = kf[kt][dc];
                wave_lds_sync();
                f32x4 s[2], dp[2];
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) {
                    s[kt] = dp[kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int dc = 0; dc < DC; ++dc) {
                        s[kt] = mma(kf[kt][dc], row.q[dc], s[kt]);
                        dp[kt] = mma(vf[kt][dc], row.d[dc], dp[kt]);
                    }
                }
                u = find(u + kWaves);
                if (u < units) fetch(u);
                const unsigned seen = p.n_buckets
                    ? score_gradients<true, true, kNarrow<T>>(p, buckets, sums, s, dp, row.lse, row.weight, row.less, row.down, far_off, offset + t0, tpt, tc, mine, now, last, g, lane)
                    : score_gradients<false, true, kNarrow<T>>(p, buckets, sums, s, dp, row.lse, row.weight, row.less, row.down, far_off, offset + t0, tpt, tc, mine, now, last, g, lane);
                V8<T> sf, rf;          // as in queries_many_kernel
                split<T>(s[0], s[1], &sf, &rf);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    const V8<T> x = transposed<T, D>(stage, dt * 16, lane);
                    if constexpr (decltype(careful)::value) {
                        acc[dt] = mma_masked<T>(x, sf, rf, seen, acc[dt]);
                    } else {
                        acc[dt] = mma(x, sf, acc[dt]);
                        if (sizeof(T) == 2) acc[dt] = mma(x, rf, acc[dt]);
                    }
                }
            }
        }
    };
    auto odd = [&]() {
        bool any = false;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) any |= not_finite(acc[dt]);
        return any;
    };
    bool again = CAREFUL;
    row.weigh(false);
    if constexpr (!CAREFUL) {
        sweep(std::false_type{});
        again = __syncthreads_or(odd());
    }
    if (again) {
        // a second time where rows are left that are not finite (they may want the smaller power of two)
        __shared__ unsigned safe;
        if (tid == 0) safe = 0;
        for (int i = 0; i < 2; ++i) {
            sweep(std::true_type{});
            if (!kNarrow<T> || i || !__syncthreads_or(odd())) break;
            if (odd()) atomicOr(&safe, 1u << c);
            __syncthreads();
            row.weigh((safe >> c) & 1);
        }
    }
    if (kNarrow<T>)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[dt] *= row.down;
    float *merge = reinterpret_cast<float *>(dynamic);
#pragma unroll
    for (int strip = 0; strip < DC; ++strip) {
        __syncthreads();               // the keys' staging, or the strip before, has been read
#pragma unroll
        for (int j = 0; j < 2; ++j) *reinterpret_cast<f32x4 *>(merge + (wave * 16 + c) * kMergeStride + 16 * j + 4 * g) = acc[2 * strip + j];
        __syncthreads();
        const int r = tid >> 3, col = (tid & 7) * 4, rt = r / p.group, t = t0 + rt;
        if (tid < 16 * 8 && rt < tpt && t < p.queries) {
            f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int x = 0; x < kWaves; ++x) sum += *reinterpret_cast<const f32x4 *>(merge + (x * 16 + r) * kMergeStride + col);
            store_row<T>(static_cast<T *>(w.dq), nullptr, (((int64_t)b * p.queries + t) * p.heads + h * p.group + (r - rt * p.group)) * D + strip * 32 + col, sum * p.scale);
        }
    }
}

template <typename T, int D>
__global__ __launch_bounds__(kThreads) void queries_few_kernel(const Problem p, const Step w, int n_tiles) {
    __shared__ List<1, kWindow> list;
    extern __shared__ __align__(16) unsigned char dynamic[];
    const int unit = xcd_contiguous_block(), pair = unit / n_tiles, tile = unit - pair * n_tiles, b = pair / p.kv_heads, h = pair - b * p.kv_heads;
    Buckets buckets;
    float *sums = nullptr;
    if (p.n_buckets) {
        unsigned char *at = dynamic + few_stage_bytes<T, D>();
        buckets = load_buckets<T>(p, h, at);
        sums = bias_place(p, at);
    }
    few_rows<T, D, false>(p, w, list, dynamic, buckets, sums + (threadIdx.x >> 6) * p.n_buckets * 64, b, h, tile, w.largest + unit);
    if (p.n_buckets) write_bias(p, sums, w.bias_sums, (int64_t)b * n_tiles + tile, h);
}

constexpr int kStep = 64;              // keys in LDS
constexpr int kListed = 256;           // blocks listed at a time

template <typename T, int D, bool BIAS> struct Steps {
    static constexpr int kKeyStride = D + kPad, kValueStride = D + 16 / sizeof(T);
    static constexpr size_t kStepBytes = (size_t)kStep * (kKeyStride + kValueStride) * sizeof(T);
    static constexpr int kBuffers = !BIAS && kStepBytes <= 40 * 1024 ? 2 : 1;     // two workgroups' worth, with the bias's sums, fits a CU's LDS
    static constexpr size_t kBytes = kBuffers * kStepBytes;
};

// RT tiles of 16 rows per wavefront, the list walked by all four together, as many_kernel does forward.
template <typename T, int D, int RT, bool BIAS>
__global__ __launch_bounds__(kThreads, 2) void queries_many_kernel(const Problem p, const Step w, int32_t *flags, int n_groups) {
    constexpr int DC = D / 32, DT = D / 16, TILES = kWaves * RT, BUFFERS = Steps<T, D, BIAS>::kBuffers;
    constexpr int KS = Steps<T, D, BIAS>::kKeyStride, VS = Steps<T, D, BIAS>::kValueStride;
    __shared__ List<TILES, kListed> list;
    __shared__ float2 tops[kWaves];
    extern __shared__ __align__(16) unsigned char dynamic[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, c = lane & 15;
    const int unit = xcd_contiguous_block(), pair = unit / n_groups, group = group_of(p, unit - pair * n_groups, n_groups), b = pair / p.kv_heads, h = pair - b * p.kv_heads;
    const int k_len = key_count(p, b), q_len = query_count(p, b), offset = k_len - q_len;
    const int tpt = tile_tokens(p.group), t0 = group * TILES * tpt;
    const int tc = c / p.group, mine = c - tc * p.group, head = h * p.group + mine;
    const bool used = tc < tpt;
    T *tiles = reinterpret_cast<T *>(dynamic);
    Buckets buckets;
    float *sums = nullptr;
    if (BIAS) {
        unsigned char *at = dynamic + Steps<T, D, BIAS>::kBytes;
        buckets = load_buckets<T>(p, h, at);
        sums = bias_place(p, at) + wave * p.n_buckets * 64;
        for (int n = 0; n < p.n_buckets; ++n) sums[n * 64 + lane] = 0.f;
    }
    Row16<T, D> row[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        row[rt].load(p, w, b, t0 + (wave * RT + rt) * tpt + tc, head, used, q_len, k_len, offset, g, true);
        row[rt].weigh(false);
    }
    if (kNarrow<T>) {
        float2 top = row[0].largest();
#pragma unroll
        for (int rt = 1; rt < RT; ++rt) {
            const float2 v = row[rt].largest();
            top = make_float2(fmaxf(top.x, v.x), fmaxf(top.y, v.y));
        }
        if (lane == 0) tops[wave] = top;
    }
    bool far_off = false;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) far_off |= BIAS && row[rt].far_off();
    const int last_key = p.causal ? min(k_len - 1, offset + min(t0 + TILES * tpt, q_len) - 1) : k_len - 1;
    const T *kbase = static_cast<const T *>(p.k) + b * p.ks.batch + h * p.ks.head;
    const T *vbase = static_cast<const T *>(p.v) + b * p.vs.batch + h * p.vs.head;
    const int sub_shift = p.block_shift - 5;

    f32x4 acc[RT][DT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[rt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int first = 0; first < p.blocks; first += kListed) {
        const int units = build_list(list, p, b, h, t0, q_len, k_len, first, min(kListed, p.blocks - first)) << sub_shift;
        auto first_key = [&](int u) {
            return __builtin_amdgcn_readfirstlane(((first + list.id[u >> sub_shift]) << p.block_shift) + ((u & ((1 << sub_shift) - 1)) << 5));
        };
        Stage<T, D> ks, vs;
        const int word = wave * RT / 4, shift = wave * RT % 4 * 16;
        int k0 = 0, k1 = 0;            // first keys of the step in the registers
        unsigned who = 0, who1 = 0;    // its tokens of the wavefront's tiles, 16 bits a tile, one word a unit
        auto tokens = [&](int u) { return u < units ? (unsigned)(list.bits[u >> sub_shift][word] >> shift) : 0u; };
        auto fetch = [&](int u) {
            k0 = first_key(u);
            k1 = u + 1 < units ? first_key(u + 1) : k0;
            ks.fetch(kbase, p.ks.row, k0, k1, k_len);
            vs.fetch(vbase, p.vs.row, k0, k1, k_len);
            who = k0 <= last_key ? tokens(u) : 0u;
            who1 = k1 <= last_key ? tokens(u + 1) : 0u;
        };
        if (units) fetch(0);
        for (int u = 0; u < units; u += 2) {
            if (BUFFERS == 1) __syncthreads();       // the step before has been read
            T *keys = BUFFERS == 2 && (u & 2) ? tiles + kStep * (KS + VS) : tiles, *values = keys + kStep * KS;
            ks.store(keys, KS);
            vs.store(values, VS);
            const int key0[2] = {k0, k1};
            constexpr unsigned ALL = RT == 2 ? ~0u : 0xffffu;
            const unsigned sel[2] = {__builtin_amdgcn_readfirstlane(who) & ALL, __builtin_amdgcn_readfirstlane(who1) & ALL};
            __syncthreads();
            if (u + 2 < units) fetch(u + 2);
#pragma unroll 1
            for (int x = 0; x < 2; ++x) {
                const unsigned bits = x ? sel[1] : sel[0];
                if (!bits) continue;                 // none of the wavefront's tokens selected the block
                const int now = x ? key0[1] : key0[0];
                const T *ktile = keys + x * kUnit * KS, *vtile = values + x * kUnit * VS;
                f32x4 s[RT][2], dp[RT][2];
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) s[rt][kt] = dp[rt][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
                    // two strips of 32 columns at a time: with all of them in registers a head of 128 spills
                    constexpr int STRIPS = DC < 2 ? DC : 2;
#pragma unroll
                    for (int d0 = 0; d0 < DC; d0 += STRIPS) {
                        V8<T> kf[STRIPS], vf[STRIPS];
#pragma unroll
                        for (int i = 0; i < STRIPS; ++i) {
                            kf[i] = load8(ktile + (kt * 16 + c) * KS + (d0 + i) * 32 + 8 * g);
                            vf[i] = load8(vtile + (kt * 16 + c) * VS + (d0 + i) * 32 + 8 * g);
                        }
#pragma unroll
                        for (int i = 0; i < STRIPS; ++i)
#pragma unroll
                            for (int rt = 0; rt < RT; ++rt) {
                                s[rt][kt] = mma(kf[i], row[rt].q[d0 + i], s[rt][kt]);
                                dp[rt][kt] = mma(vf[i], row[rt].d[d0 + i], dp[rt][kt]);
                            }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
                // the first columns of the keys are read while the powers are taken
                constexpr int XB = DT < 4 ? DT / 2 : DT / 4;
                V8<T> xf[XB];
                auto read_keys = [&](int part) {
#pragma unroll
                    for (int i = 0; i < XB; ++i) xf[i] = transposed<T, D>(ktile, (part * XB + i) * 16, lane);
                };
                read_keys(0);
                __builtin_amdgcn_sched_barrier(0);
                bool edge = false;
                float lse[RT];
                int last[RT];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    // a row that did not select the block has its powers relative to +inf: 0
                    const bool one = !used || (bits >> (16 * rt + tc)) & 1;
                    lse[rt] = one ? row[rt].lse : __builtin_inff();
                    last[rt] = one ? row[rt].limit : -1;
                    edge |= one && now + kUnit - 1 > row[rt].limit;
                }
                const int pos = offset + t0 + wave * RT * tpt;
                if (__any(edge)) {
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                        score_gradients<BIAS, true, kNarrow<T>>(p, buckets, sums, s[rt], dp[rt], lse[rt], row[rt].weight, row[rt].less, row[rt].down, far_off, pos + rt * tpt, tpt, tc, mine, now, last[rt], g, lane);
                } else {
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                        score_gradients<BIAS, false, kNarrow<T>>(p, buckets, sums, s[rt], dp[rt], lse[rt], row[rt].weight, row[rt].less, row[rt].down, far_off, pos + rt * tpt, tpt, tc, mine, now, 0, g, lane);
                }
                // dS goes into the product with K rounded, and what that took (in 16 bits) in a second one: a row's dS add up to 0, and its keys
                // have much in common, so that the rounding alone would be larger than dQ's own
                V8<T> sf[RT], rf[RT];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) split<T>(s[rt][0], s[rt][1], &sf[rt], &rf[rt]);
#pragma unroll
                for (int part = 0; part < DT / XB; ++part) {
#pragma unroll
                    for (int i = 0; i < XB; ++i)
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt) {
                            acc[rt][part * XB + i] = mma(xf[i], sf[rt], acc[rt][part * XB + i]);
                            if (sizeof(T) == 2) acc[rt][part * XB + i] = mma(xf[i], rf[rt], acc[rt][part * XB + i]);
                        }
                    if (part + 1 < DT / XB) read_keys(part + 1);
                }
            }
        }
    }
    bool odd = false;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int t = t0 + (wave * RT + rt) * tpt + tc;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            odd |= not_finite(acc[rt][dt]);
            if (used && t < p.queries)
                store_row<T>(static_cast<T *>(w.dq), nullptr, (((int64_t)b * p.queries + t) * p.heads + head) * D + dt * 16 + 4 * g,
                             acc[rt][dt] * (kNarrow<T> ? p.scale * row[rt].down : p.scale));
        }
    }
    if (BIAS) write_bias(p, sums - wave * p.n_buckets * 64, w.bias_sums, (int64_t)b * n_groups + group, h);
    odd = __syncthreads_or(odd);
    if (tid == 0) {
        flags[unit] = odd;
        if (kNarrow<T>) {
            float2 top = tops[0];
            for (int i = 1; i < kWaves; ++i) top = make_float2(fmaxf(top.x, tops[i].x), fmaxf(top.y, tops[i].y));
            w.largest[unit] = top;
        }
    }
}

// The tiles of queries_many_kernel's workgroups with a result that was not finite, again.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void queries_redo_kernel(const Problem p, const Step w, const int32_t *flags, int n_groups, int tiles) {
    __shared__ List<1, kWindow> list;
    extern __shared__ __align__(16) unsigned char dynamic[];
    const int unit = xcd_contiguous_block();
    if (!flags[unit]) return;
    const int pair = unit / n_groups, group = group_of(p, unit - pair * n_groups, n_groups), b = pair / p.kv_heads, h = pair - b * p.kv_heads;
    Buckets buckets;
    float *sums = nullptr;
    if (p.n_buckets) {
        unsigned char *at = dynamic + few_stage_bytes<T, D>();
        buckets = load_buckets<T>(p, h, at);
        sums = bias_place(p, at);
    }
    for (int i = 0; i < tiles; ++i) {
        __syncthreads();               // the joining buffer and the bias's sums of the tile before have been read
        few_rows<T, D, true>(p, w, list, dynamic, buckets, sums + (threadIdx.x >> 6) * p.n_buckets * 64, b, h, group * tiles + i, nullptr);
        if (p.n_buckets) write_bias(p, sums, w.bias_sums, (int64_t)b * n_groups + group, h, i > 0);
    }
}

// dbias[n, head]: the tiles' sums in order, a share of them for each group of threads, then the shares in order.
template <typename T>
__global__ __launch_bounds__(1024) void bias_kernel(const float *sums, T *dbias, int tiles, int heads, int n_buckets) {
    __shared__ float shares[1024];
    const int head = blockIdx.x, parts = 1024 / n_buckets, n = threadIdx.x % n_buckets, part = threadIdx.x / n_buckets;
    float total = 0.f;
    if (part < parts)
        for (int t = part; t < tiles; t += parts) total += sums[((int64_t)t * heads + head) * n_buckets + n];
    shares[threadIdx.x] = total;
    __syncthreads();
    if (part == 0) {
        for (int x = 1; x < parts; ++x) total += shares[x * n_buckets + n];
        dbias[(int64_t)n * heads + head] = (T)total;
    }
}

// ---- by block: dK and dV ----------------------------------------------------------------------------------

template <typename T, int D> constexpr size_t keys_stage_bytes() { return (size_t)kWaves * 2 * kUnit * (D + kPad) * sizeof(T); }

// A wavefront has KT tiles of 16 keys; where a block has fewer than four wavefronts' keys, several share them and take the list's rows in turn.
// flags[workgroup]: whether a sum was not finite; CAREFUL: those again, with such places apart.
template <typename T, int D> struct Keys {
    // heads of 128: two tiles' operands and sums leave room for one wavefront per SIMD alone, and still take less than one tile each of two
    // wavefronts that fetch and turn every row for half the keys (2 x 4,096 tokens, 16 / 4 heads 371 and 565 us, either with one product less)
    static constexpr int kTiles = sizeof(T) == 4 ? 1 : 2;
    static constexpr int kResident = D == 128 ? 1 : 2;
    // neighbouring lanes fetch neighbouring 16 bytes of a row, and the operands are read from LDS: a third of the accesses that lanes with rows of
    // their own, as the operands lie, make (8,192 tokens, 16 / 1 heads of 64 171 and 191 us).  With heads of 128, where a wavefront is
    // alone, the way through LDS costs more than that (2 x 4,096 tokens, 16 / 4 heads 406 and 344 us).
    static constexpr bool kAlong = D != 128;
    static int parts(int block) { return std::max(1, block / (kWaves * 16 * kTiles)); }       // workgroups of a block
};

template <typename T, int D, bool CAREFUL>
__global__ __launch_bounds__(kThreads, (Keys<T, D>::kResident)) void keys_kernel(const Problem p, const T *dout, Strides ds, const float2 *lse, const float *delta, const float2 *tops, int n_tops, const Piece *pieces,
                                                        const int32_t *totals, const int32_t *count, const int32_t *list, float *partial, T *dk, T *dv, int32_t *flags) {
    constexpr int DC = D / 32, DT = D / 16, S = D + kPad, KT = Keys<T, D>::kTiles;
    constexpr int EPC = 16 / sizeof(T), CPR = D / EPC, RPL = 64 / CPR, N = kUnit / RPL;
    constexpr bool ALONG = Keys<T, D>::kAlong;
    struct Row { float lse, delta; int pos, head; };
    __shared__ Row rows[kWaves][kUnit];
    __shared__ float mores[kWaves][kUnit];
    extern __shared__ __align__(16) unsigned char dynamic[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, c = lane & 15;
    const int block = 1 << p.block_shift, kw_n = min(kWaves, block / (16 * KT)), rw_n = kWaves / kw_n, parts = block / (kw_n * 16 * KT);
    const int kw = wave % kw_n, rw = wave / kw_n;
    // (dealt to the XCDs in turn: contiguous shares, for the L2s' sake, are uneven and take 4 to 15 % more)
    const int unit = blockIdx.x, work = unit / parts, part = unit - work * parts;
    if ((!count && work >= totals[0] + p.batch * p.kv_heads * p.blocks) || (CAREFUL && !flags[unit])) return;
    const Piece piece = count ? Piece{work, work * p.queries, count[work], -1} : pieces[work];      // short lists have a place each
    if (piece.len < 0) return;
    const int pair = piece.block / p.blocks, blk = piece.block - pair * p.blocks, b = pair / p.kv_heads, h = pair - b * p.kv_heads;
    const int k_len = key_count(p, b), q_len = query_count(p, b), offset = k_len - q_len;
    const int in_block = (part * kw_n + kw) * 16 * KT, key0 = (blk << p.block_shift) + in_block, n_rows = piece.len * p.group;

    T *stage_q = reinterpret_cast<T *>(dynamic) + wave * 2 * kUnit * S, *stage_d = stage_q + kUnit * S;
    Buckets buckets;
    if (p.n_buckets) {
        buckets = load_buckets<T>(p, h, dynamic + keys_stage_bytes<T, D>());
        __syncthreads();
    }

    V8<T> kf[KT][DC], vf[KT][DC];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
        const int key = key0 + kt * 16 + c;
        const bool there = key < k_len;
        const T *ks = static_cast<const T *>(p.k) + b * p.ks.batch + h * p.ks.head + (int64_t)key * p.ks.row + 8 * g;
        const T *vs = static_cast<const T *>(p.v) + b * p.vs.batch + h * p.vs.head + (int64_t)key * p.vs.row + 8 * g;
#pragma unroll
        for (int dc = 0; dc < DC; ++dc) {
            kf[kt][dc] = there ? load8(ks + dc * 32) : zero8<T>();
            vf[kt][dc] = there ? load8(vs + dc * 32) : zero8<T>();
        }
    }
    const T *qbase = static_cast<const T *>(p.q) + b * p.qs.batch + (int64_t)h * p.group * p.qs.head + (ALONG ? lane % CPR * EPC : 8 * g);
    const T *dbase = dout + b * ds.batch + (int64_t)h * p.group * ds.head + (ALONG ? lane % CPR * EPC : 8 * g);
    Row *own = rows[wave];
    // Logarithms of the rows' sums, where they are not added to the references: with a bias, whose scores are formed apart from them as the forward
    // pass does, and in steps with a reference so large that the sum would lose its last bits (from 2^24 on all of it).
    float *more = mores[wave];

    // float16: powers are 2^kGain times p, so that shares of one in a million keep their bits, and dS is 2^kGain gain p (dP - delta) with a
    // power of two that keeps gain (|dO| |V| + |delta|), a bound on gain |dP - delta|, below 2^4.  It goes by the longest of this wavefront's
    // values and the largest rows of the sequence's heads, of those that are finite.  (A gain that follows the rows of the list,
    // reducing the sums when a larger one comes, takes 24 us more of 8,192 tokens' 176, this 7.  p may pass 1 by what rounding does to
    // large scores.)
    constexpr int kGain = kNarrow<T> ? 10 : 0;
    float gain = 1.f;
    if constexpr (kNarrow<T>) {
        float longest = 0.f;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
            float squares = 0.f;
#pragma unroll
            for (int dc = 0; dc < DC; ++dc)
#pragma unroll
                for (int i = 0; i < 8; ++i) squares += (float)vf[kt][dc][i] * (float)vf[kt][dc][i];
            squares = rows_sum(squares);
            longest = fmaxf(longest, squares < __builtin_inff() ? squares : 0.f);
        }
        float2 top = make_float2(0.f, 0.f);
#pragma unroll 4
        for (int i = tid; i < n_tops; i += kThreads) {
            const float2 v = tops[(int64_t)pair * n_tops + i];
            top = make_float2(fmaxf(top.x, v.x), fmaxf(top.y, v.y));
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            longest = fmaxf(longest, __shfl_xor(longest, d));
            top.x = fmaxf(top.x, __shfl_xor(top.x, d));
            top.y = fmaxf(top.y, __shfl_xor(top.y, d));
        }
        if (lane < 2) mores[wave][lane] = lane ? top.y : top.x;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kWaves; ++i) top = make_float2(fmaxf(top.x, mores[i][0]), fmaxf(top.y, mores[i][1]));
        gain = __builtin_amdgcn_ldexpf(16.f, -__builtin_amdgcn_frexp_expf(top.x * __builtin_sqrtf(longest) + top.y));
        __syncthreads();
    }

    f32x4 ak[KT][DT], av[KT][DT];
    {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) ak[kt][dt] = av[kt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
        u32x4 qr[N], dr[N];            // rows as they lie in memory, or
        V8<T> qf[2][DC], df[2][DC];    // operands
        float next_more = 0.f;
        Row next;                      // lane r, up to 31: row r of the step
        // the lane's row (lane & 31) of the step that is fetched next: place in the list, head, and the token, whose load has a step's time
        // before the rows' own depend on it
        const int stride = rw_n * kUnit, places = stride / p.group, heads = stride - places * p.group;
        int r0 = rw * kUnit, at = (r0 + (lane & 31)) / p.group, x = r0 + (lane & 31) - at * p.group, token = 0;
        auto look = [&]() { token = list[piece.start + min(at, piece.len - 1)]; };
        // rows behind the last read it again, and have no weight
        auto fetch = [&]() {
            const int64_t row = ((int64_t)b * p.queries + token) * p.heads + h * p.group + x;
            const float2 ls = lse[row];
            next = Row{ls.x, delta[row], offset + token, x};
            next_more = ls.y - kGain;
            if (at >= piece.len) {
                next.lse = __builtin_inff();
                next.delta = next_more = 0.f;
            }
            if constexpr (ALONG) {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int t = __shfl(token, i * RPL + lane / CPR), y = __shfl(x, i * RPL + lane / CPR);
                    qr[i] = *reinterpret_cast<const u32x4 *>(qbase + (int64_t)t * p.qs.row + y * p.qs.head);
                    dr[i] = *reinterpret_cast<const u32x4 *>(dbase + (int64_t)t * ds.row + y * ds.head);
                }
            } else {
#pragma unroll
                for (int rt = 0; rt < 2; ++rt) {
                    const int t = __shfl(token, rt * 16 + c), y = __shfl(x, rt * 16 + c);
                    const T *q = qbase + (int64_t)t * p.qs.row + y * p.qs.head, *d = dbase + (int64_t)t * ds.row + y * ds.head;
#pragma unroll
                    for (int dc = 0; dc < DC; ++dc) {
                        qf[rt][dc] = load8(q + dc * 32);
                        df[rt][dc] = load8(d + dc * 32);
                    }
                }
            }
            at += places;
            x += heads;
            if (x >= p.group) { x -= p.group; ++at; }
        };
        if (r0 < n_rows) {
            look();
            fetch();
            look();
        }
        while (r0 < n_rows) {
            wave_lds_sync();
            if constexpr (ALONG) {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int to = (i * RPL + lane / CPR) * S + lane % CPR * EPC;
                    *reinterpret_cast<u32x4 *>(stage_q + to) = qr[i];
                    *reinterpret_cast<u32x4 *>(stage_d + to) = dr[i];
                }
            } else {
#pragma unroll
                for (int rt = 0; rt < 2; ++rt)
#pragma unroll
                    for (int dc = 0; dc < DC; ++dc) {
                        *reinterpret_cast<V8<T> *>(stage_q + (rt * 16 + c) * S + dc * 32 + 8 * g) = qf[rt][dc];
                        *reinterpret_cast<V8<T> *>(stage_d + (rt * 16 + c) * S + dc * 32 + 8 * g) = df[rt][dc];
                    }
            }
            const bool apart = p.n_buckets || __any(fabsf(next.lse) > 4096.f && next.lse < __builtin_inff());
            if (!apart) next.lse += next_more;
            if (kNarrow<T>) next.delta *= gain;
            if (lane < kUnit) {
                own[lane] = next;
                if (apart) more[lane] = next_more;
            }
            wave_lds_sync();
            // tokens ascend
            const int from = __builtin_amdgcn_readfirstlane(next.pos), to = __builtin_amdgcn_readlane(next.pos, kUnit - 1);
            r0 += stride;
            if (ALONG) {
                fetch();
                look();
            }
            f32x4 s[2][KT], dp[2][KT];  // [rows][keys]
#pragma unroll
            for (int rt = 0; rt < 2; ++rt) {
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) s[rt][kt] = dp[rt][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int dc = 0; dc < DC; ++dc) {
                    V8<T> q, d;
                    if constexpr (ALONG) {
                        q = load8(stage_q + (rt * 16 + c) * S + dc * 32 + 8 * g);
                        d = load8(stage_d + (rt * 16 + c) * S + dc * 32 + 8 * g);
                    } else {
                        q = qf[rt][dc];
                        d = df[rt][dc];
                    }
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt) {
                        s[rt][kt] = mma(q, kf[kt][dc], s[rt][kt]);
                        dp[rt][kt] = mma(d, vf[kt][dc], dp[rt][kt]);
                    }
                }
            }
            if (!ALONG) {
                fetch();
                look();
            }

            unsigned seen[KT] = {};
            auto gradients = [&](auto masked) {
#pragma unroll
                for (int rt = 0; rt < 2; ++rt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const Row row = own[rt * 16 + 4 * g + i];
#pragma unroll
                        for (int kt = 0; kt < KT; ++kt) {
                            const float z = apart ? s[rt][kt][i] : s[rt][kt][i] * p.scale2 - row.lse;
                            float y = __builtin_amdgcn_exp2f(z);
                            float e = y * (kNarrow<T> ? dp[rt][kt][i] * gain - row.delta : dp[rt][kt][i] - row.delta);
                            if constexpr (decltype(masked)::value) {
                                const int key = key0 + kt * 16 + c;
                                const bool ok = key <= (p.causal ? row.pos : k_len - 1) && (!CAREFUL || row.lse < __builtin_inff());
                                y = ok ? y : 0.f;
                                e = ok ? e : 0.f;
                                seen[kt] |= (unsigned)ok << (4 * rt + i);
                            }
                            s[rt][kt][i] = y;
                            dp[rt][kt][i] = e;
                        }
                    }
            };
            if (p.n_buckets) {
                const int near = buckets.at(from - (key0 + 16 * KT - 1)), far = buckets.at(to - key0);
#pragma unroll
                for (int rt = 0; rt < 2; ++rt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const Row row = own[rt * 16 + 4 * g + i];
                        const float less = more[rt * 16 + 4 * g + i], same = near == far ? buckets.value(near, row.head) : 0.f;
#pragma unroll
                        for (int kt = 0; kt < KT; ++kt) {
                            float z = s[rt][kt][i] * p.scale2 + same;
                            if (near != far) z += buckets.value(buckets.at(row.pos - (key0 + kt * 16 + c)), row.head);
                            s[rt][kt][i] = (z - row.lse) - less;
                        }
                    }
            } else if (apart) {
#pragma unroll
                for (int rt = 0; rt < 2; ++rt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float lse = own[rt * 16 + 4 * g + i].lse, less = more[rt * 16 + 4 * g + i];
#pragma unroll
                        for (int kt = 0; kt < KT; ++kt) s[rt][kt][i] = __builtin_fmaf(s[rt][kt][i], p.scale2, -lse) - less;
                    }
            }
            if (CAREFUL || key0 + 16 * KT > k_len || (p.causal && from < key0 + 16 * KT - 1)) gradients(std::true_type{});
            else gradients(std::false_type{});
            // the powers go into dV's product rounded, and what that took (in 16 bits) in a second one: nearly even ones are all rounded the
            // same way, which no sum evens out (2 x 4,096 tokens, 16 / 4 heads 27 us); so does dS into dK's, whose error would be 1.4 times that
            // of rounding dK itself (22 us)
            V8<T> pf[KT], pl[KT], sf[KT], sl[KT];
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                split<T>(s[0][kt], s[1][kt], &pf[kt], &pl[kt]);
                split<T>(dp[0][kt], dp[1][kt], &sf[kt], &sl[kt]);
            }
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const V8<T> d = transposed<T, D>(stage_d, dt * 16, lane), q = transposed<T, D>(stage_q, dt * 16, lane);
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    if constexpr (CAREFUL) {
                        av[kt][dt] = mma_masked<T>(d, pf[kt], pl[kt], seen[kt], av[kt][dt]);
                        ak[kt][dt] = mma_masked<T>(q, sf[kt], sl[kt], seen[kt], ak[kt][dt]);
                    } else {
                        av[kt][dt] = mma(d, pf[kt], av[kt][dt]);
                        if (sizeof(T) == 2) av[kt][dt] = mma(d, pl[kt], av[kt][dt]);
                        ak[kt][dt] = mma(q, sf[kt], ak[kt][dt]);
                        if (sizeof(T) == 2) ak[kt][dt] = mma(q, sl[kt], ak[kt][dt]);
                    }
                }
            }
        }
    }
    bool odd = false;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) odd |= not_finite(ak[kt][dt]) || not_finite(av[kt][dt]);
    if (!CAREFUL) {
        odd = __syncthreads_or(odd);
        if (tid == 0) flags[unit] = odd;
    }

    if constexpr (kNarrow<T>) {
        const float share = 1.f / (1 << kGain);
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) { ak[kt][dt] *= share / gain; av[kt][dt] *= share; }
    }

    // wavefronts that share keys: the upper half hands its sums to the lower one, until one has them all
    f32x4 *merge = reinterpret_cast<f32x4 *>(dynamic);
    for (int half = rw_n >> 1; half; half >>= 1) {
        __syncthreads();
        if (rw >= half && rw < 2 * half) {
            f32x4 *to = merge + ((rw - half) * kw_n + kw) * (2 * KT * DT * 64) + lane;
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) { to[(kt * DT + dt) * 128] = ak[kt][dt]; to[(kt * DT + dt) * 128 + 64] = av[kt][dt]; }
        }
        __syncthreads();
        if (rw < half) {
            const f32x4 *from = merge + (rw * kw_n + kw) * (2 * KT * DT * 64) + lane;
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) { ak[kt][dt] += from[(kt * DT + dt) * 128]; av[kt][dt] += from[(kt * DT + dt) * 128 + 64]; }
        }
    }
    if (rw) return;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
        const int key = key0 + kt * 16 + c;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            const int d = dt * 16 + 4 * g;
            if (piece.slot >= 0) {
                float *to = partial + ((int64_t)piece.slot * 2 * block + in_block + kt * 16 + c) * D + d;
                *reinterpret_cast<f32x4 *>(to) = ak[kt][dt];
                *reinterpret_cast<f32x4 *>(to + (int64_t)block * D) = av[kt][dt];
            } else if (key < p.keys) {
                const int64_t at = (((int64_t)b * p.keys + key) * p.kv_heads + h) * D + d;
#pragma unroll
                for (int i = 0; i < 4; ++i) { dk[at + i] = (T)(ak[kt][dt][i] * p.scale); dv[at + i] = (T)av[kt][dt][i]; }
            }
        }
    }
}

// Blocks whose lists were cut: the pieces' sums, in order, four columns of a key a thread.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void pieces_kernel(const Problem p, const int32_t *count, const int32_t *slot0, const float *partial, T *dk, T *dv, int piece) {
    const int block = 1 << p.block_shift, each = 2 * block * (D / 4) / kThreads;       // a multiple of kThreads: blocks of 32 and more, heads of 32 and more
    const int m = blockIdx.x / each, k = (count[m] + piece - 1) / piece;
    if (k <= 1) return;
    const int pair = m / p.blocks, blk = m - pair * p.blocks, b = pair / p.kv_heads, h = pair - b * p.kv_heads;
    const int e = (blockIdx.x - m * each) * kThreads + threadIdx.x, row = e / (D / 4), col = (e - row * (D / 4)) * 4, key = (blk << p.block_shift) + (row & (block - 1));
    if (key >= p.keys) return;
    const float *src = partial + ((int64_t)slot0[m] * 2 * block + row) * D + col;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    each_piece(0, k, [&](int i) { return *reinterpret_cast<const f32x4 *>(src + (int64_t)i * 2 * block * D); }, [&](int, f32x4 v) { sum += v; });
    store_row<T>(row < block ? dk : dv, nullptr, (((int64_t)b * p.keys + key) * p.kv_heads + h) * D + col, sum * (row < block ? p.scale : 1.f));
}

// ---- host -------------------------------------------------------------------------------------------------

struct Layout {
    bool many, short_lists;
    int n_groups, chunks, piece;               // n_groups: workgroups per sequence and key head of the sweep by query
    int64_t all, pieces, slots, entries;       // blocks of all sequences and key heads; bounds on the others
    size_t delta, largest, flags, bits, count, offset, piece0, slot0, totals, list, table, partial, bias, bytes;
};

int layout_of(const Problem &p, int head_len, int row_tiles, int parts, bool narrow, Layout *l) {
    const int tpt = tile_tokens(p.group), block = 1 << p.block_shift;
    const int64_t pairs = (int64_t)p.batch * p.kv_heads;
    auto tiles = [&](int n) { return (p.queries + n * tpt - 1) / (n * tpt); };
    // as the forward pass decides it; a whole step with the kernels for few / many queries: 1,024 tokens of 32 / 8 heads of 128 in bfloat16 (256
    // workgroups) 326 / 225 us, 2,048 788 / 403; 2 x 1,024 tokens of 8 / 8 heads of 64 in 32 bits 207 / 221, 2 x 2,048 387 / 371
    l->n_groups = tiles(kWaves * row_tiles);
    l->many = pairs * l->n_groups >= 256 && 2 * p.queries >= kWaves * row_tiles * tpt;
    if (!l->many) l->n_groups = tiles(1);
    l->chunks = std::max(1, (p.queries + 63) / 64);
    // a block's list is cut into pieces of 768 to 2,048 rows (tokens times heads of the group), some 1,024 pieces in all, or of 512 where those
    // would not fill the CUs: longer ones leave CUs idle, shorter ones write more sums (of the largest calls longer ones, so that the sums
    // need not much more memory than the gradients). All of the keys' gradients with pieces of 1,024 / 1,536 / 2,048 rows: 2 x 2,048 tokens of 16 / 4 heads of 128 186 / 190 /
    // 219 us, 8,192 of 16 / 1 heads of 64 216 / 217 / 248, 2 x 4,096 of 16 / 4 heads of 128 410 / 398 / 396; a whole step of 1,070
    // tokens x 2 heads of 128 in 32 bits with 256 / 512 / 768: 178 / 164 / 211
    const int64_t rows = pairs * p.queries * std::min(p.topk, p.blocks) * p.group;
    l->piece = (int)std::max<int64_t>(1, std::min(std::max<int64_t>(2048, rows / 8192), std::max<int64_t>(rows < 256 * 768 ? 512 : 768, rows / 1024)) / p.group);
    l->all = pairs * p.blocks;
    // short lists: one kernel instead of five, whose looks through the selections stay below their launches' time
    l->short_lists = (int64_t)p.queries * p.group <= 768 && (int64_t)p.queries * p.topk <= 4096;
    l->entries = l->short_lists ? l->all * p.queries : pairs * p.queries * std::min(p.topk, p.blocks);
    l->pieces = l->short_lists ? l->all : l->all + l->entries / l->piece;
    // a list of n tokens that is cut has floor(n / piece) + 1 pieces at most, and no more than 2 floor(n / piece)
    l->slots = l->short_lists || p.queries <= l->piece ? 0 : std::min(2 * (l->entries / l->piece), l->entries / l->piece + l->all);
    const int64_t limit = INT32_MAX;
    if (l->entries > limit || l->pieces * parts > limit || l->all * (2 * block * head_len / 4 / kThreads) > limit || pairs * std::max(l->n_groups, l->chunks) > limit)
        return fail(FG_ERR_SHAPE, "block attention gradients: %lld selections of %lld blocks do not fit the 32-bit lists", (long long)l->entries, (long long)l->all);
    size_t at = 0;
    auto place = [&](size_t n) { const size_t here = at; at += (n + 255) & ~(size_t)255; return here; };
    l->delta = place((size_t)p.batch * p.queries * p.heads * sizeof(float));
    l->largest = place(narrow ? (size_t)pairs * l->n_groups * sizeof(float2) : 0);
    l->flags = place((size_t)std::max(pairs * l->n_groups, l->pieces * parts) * sizeof(int32_t));
    l->bits = place(l->short_lists ? 0 : (size_t)l->all * l->chunks * 8);
    l->count = place((size_t)l->all * 4);
    l->offset = place((size_t)l->all * 4);
    l->piece0 = place((size_t)l->all * 4);
    l->slot0 = place((size_t)l->all * 4);
    l->totals = place(4);
    l->list = place((size_t)l->entries * 4);
    l->table = place(l->short_lists ? 0 : (size_t)l->pieces * sizeof(Piece));
    l->partial = place((size_t)l->slots * 2 * block * head_len * sizeof(float));
    l->bias = place((size_t)p.batch * l->n_groups * p.heads * p.n_buckets * sizeof(float));
    l->bytes = at;
    return FG_OK;
}

template <typename T, int D>
int launch(const Problem &p, const fg_block_attention_args *a, const fg_block_attention_grads *grads, void *workspace, size_t bytes, size_t *need, hipStream_t stream) {
    constexpr int RT = sizeof(T) == 4 ? 1 : 2;
    Layout l;
    const int block = 1 << p.block_shift, parts = Keys<T, D>::parts(block);
    if (int rc = layout_of(p, D, RT, parts, kNarrow<T>, &l)) return rc;
    if (need) { *need = l.bytes; return FG_OK; }
    if (bytes < l.bytes || (l.bytes && !workspace)) return fail(FG_ERR_ARG, "block attention gradients: a workspace of %zu bytes, %zu needed (fg_block_attention_backward_workspace)", bytes, l.bytes);
    Strides ds;
    if (int rc = strides_of("dout", grads->dout, grads->dout_strides, sizeof(T), &ds)) return rc;
    unsigned char *w = static_cast<unsigned char *>(workspace);
    auto ints = [&](size_t at) { return reinterpret_cast<int32_t *>(w + at); };
    auto floats = [&](size_t at) { return reinterpret_cast<float *>(w + at); };
    const Step step{grads->dout, a->out, a->rest, ds, reinterpret_cast<const float2 *>(a->lse), floats(l.delta), reinterpret_cast<float2 *>(w + l.largest), grads->dq, floats(l.bias)};
    const dim3 threads(kThreads);
    if (p.queries && p.batch) {
        const dim3 blocks((unsigned)(p.batch * p.kv_heads * l.n_groups));
        const size_t few = few_stage_bytes<T, D>() + bias_bytes(p);
        if (l.many) {
            if (p.n_buckets) queries_many_kernel<T, D, RT, true><<<blocks, threads, Steps<T, D, true>::kBytes + bias_bytes(p), stream>>>(p, step, ints(l.flags), l.n_groups);
            else queries_many_kernel<T, D, RT, false><<<blocks, threads, Steps<T, D, false>::kBytes, stream>>>(p, step, ints(l.flags), l.n_groups);
            FG_HIP_TRY(hipGetLastError());
            queries_redo_kernel<T, D><<<blocks, threads, few, stream>>>(p, step, ints(l.flags), l.n_groups, kWaves * RT);
        } else {
            queries_few_kernel<T, D><<<blocks, threads, few, stream>>>(p, step, l.n_groups);
        }
        FG_HIP_TRY(hipGetLastError());
    }
    if (p.n_buckets && grads->dbias) {
        bias_kernel<T><<<dim3(p.heads), dim3(1024), 0, stream>>>(floats(l.bias), static_cast<T *>(grads->dbias), p.batch * l.n_groups, p.heads, p.n_buckets);
        FG_HIP_TRY(hipGetLastError());
    }
    if (!grads->dk || l.all == 0) return FG_OK;
    auto bits = reinterpret_cast<unsigned long long *>(w + l.bits);
    auto pieces = reinterpret_cast<Piece *>(w + l.table);
    const int all = (int)l.all, per_wave = (all + kWaves - 1) / kWaves;
    if (l.short_lists) {
        short_lists_kernel<<<dim3(per_wave), threads, 0, stream>>>(p, ints(l.count), ints(l.list), all);
    } else {
        mark_kernel<<<dim3((unsigned)(p.batch * p.kv_heads * l.chunks)), threads, 0, stream>>>(p, bits, l.chunks);
        count_kernel<<<dim3(per_wave), threads, 0, stream>>>(bits, ints(l.count), all, p.blocks, l.chunks);
        scan_kernel<<<dim3(1), dim3(kScan), 0, stream>>>(ints(l.count), ints(l.offset), ints(l.piece0), ints(l.slot0), ints(l.totals), all, l.piece);
        fill_kernel<<<dim3(per_wave), threads, 0, stream>>>(bits, ints(l.count), ints(l.offset), ints(l.piece0), ints(l.slot0), ints(l.totals), ints(l.list), pieces, all, p.blocks, l.chunks, l.piece);
    }
    FG_HIP_TRY(hipGetLastError());
    const size_t lds = keys_stage_bytes<T, D>() + buckets_bytes(p.n_buckets, p.low, p.high, p.group);
    auto keys = [&](auto kernel) {
        kernel<<<dim3((unsigned)(l.pieces * parts)), threads, lds, stream>>>(p, static_cast<const T *>(grads->dout), ds, reinterpret_cast<const float2 *>(a->lse), floats(l.delta), step.largest, l.n_groups, pieces, ints(l.totals),
                                                                             l.short_lists ? ints(l.count) : nullptr, ints(l.list),
                                                                             floats(l.partial), static_cast<T *>(grads->dk), static_cast<T *>(grads->dv), ints(l.flags));
    };
    keys(keys_kernel<T, D, false>);
    FG_HIP_TRY(hipGetLastError());
    keys(keys_kernel<T, D, true>);
    if (l.slots)
        pieces_kernel<T, D><<<dim3((unsigned)(all * (2 * block * (D / 4) / kThreads))), threads, 0, stream>>>(p, ints(l.count), ints(l.slot0), floats(l.partial), static_cast<T *>(grads->dk),
                                                                                                            static_cast<T *>(grads->dv), l.piece);
    FG_HIP_TRY(hipGetLastError());
    return FG_OK;
}

template <typename T> int launch_d(const Problem &p, const fg_block_attention_args *a, const fg_block_attention_grads *g, void *w, size_t bytes, size_t *need, hipStream_t stream) {
    switch (a->head_len) {
    case 32: return launch<T, 32>(p, a, g, w, bytes, need, stream);
    case 64: return launch<T, 64>(p, a, g, w, bytes, need, stream);
    default: return launch<T, 128>(p, a, g, w, bytes, need, stream);
    }
}

int launch_t(const Problem &p, const fg_block_attention_args *a, const fg_block_attention_grads *g, void *w, size_t bytes, size_t *need, hipStream_t stream) {
    switch (a->type) {
    case FG_TYPE_F32: return launch_d<float>(p, a, g, w, bytes, need, stream);
    case FG_TYPE_F16: return launch_d<_Float16>(p, a, g, w, bytes, need, stream);
    default: return launch_d<__bf16>(p, a, g, w, bytes, need, stream);
    }
}
}  // namespace
}  // namespace block
}  // namespace fg

extern "C" int64_t fg_block_attention_backward_workspace(const fg_block_attention_args *args) {
    fg::block::Problem p;
    if (int rc = fg::block::problem_of(args, &p)) return rc;
    size_t need = 0;
    const int rc = fg::block::launch_t(p, args, nullptr, nullptr, 0, &need, nullptr);
    return rc ? rc : (int64_t)need;
}

extern "C" int fg_block_attention_backward(const fg_block_attention_args *args, const fg_block_attention_grads *grads, void *workspace,
                                           size_t workspace_bytes, void *stream) {
    fg::block::Problem p;
    if (int rc = fg::block::problem_of(args, &p)) return rc;
    if (!grads) return fg::fail(FG_ERR_ARG, "block attention gradients: null pointer");
    if (p.batch && ((p.queries && (!p.q || !p.list || !args->out || !args->lse || !grads->dout || !grads->dq)) || (p.keys && (!p.k || !p.v)) ||
        !grads->dk != !grads->dv || (p.n_buckets && !p.bias)))
        return fg::fail(FG_ERR_ARG, "block attention gradients: null pointer");
    using fg::block::aligned;
    int rc;
    if ((rc = aligned("the workspace", workspace, 16)) || (rc = aligned("dq", grads->dq, 16)) || (rc = aligned("dk", grads->dk, 16)) ||
        (rc = aligned("dv", grads->dv, 16)) || (rc = aligned("dbias", grads->dbias, args->type == FG_TYPE_F32 ? 4 : 2))) return rc;
    return fg::block::launch_t(p, args, grads, workspace, workspace_bytes, nullptr, static_cast<hipStream_t>(stream));
}
