// Softmax attention over the blocks of keys that every query selected, forward:
//   out[i, h] = sum_j p_ij V[j, g],  p_i = softmax over the visible keys j of  scale <Q[i, h], K[j, g]> + bias[bucket(pos_i - j), h]
// with g = h / group, pos_i = k_len - q_len + i, and j visible to i where floor(j / block) is in i's list for g, j < k_len and (causal) j <= pos_i.
// No visible key: 0.
//
// Rows of one token's heads and of neighbouring tokens make tiles of 16, and the blocks that any token of a tile selected are walked for all of
// them; a token that did not select one has weight 0 there.  That pays as far as neighbours select the same blocks: 8,192 tokens, 32 / 8
// heads of 128, 16 blocks of 64 take 373 us where they look for what a stretch of 128 tokens looks for, and 661 where every one draws its
// own.  Two kernels.
// many_kernel, where there are queries to fill the card: four wavefronts with tiles of their own walk the union of their lists through
// LDS, 64 keys at a time, fetched into registers while the 64 before are worked on; each keeps its softmax and its output.
// few_kernel, for single tokens and short sequences: one tile per workgroup, whose list is dealt out to the four wavefronts and, where
// that leaves the card idle, to several workgroups; each takes its keys from memory straight into operands.
// Values that are not finite reach the rows that see them and no others: a result that is not finite is computed again with such places
// apart (mma_masked).
//
// What bounds them.  many_kernel, those 8,192 tokens in bfloat16: 406 us, 320 TFLOP/s of the selected pairs;
// the matrix cores are busy a fifth of the time, for unions are larger than their tokens' lists, 256 registers allow two wavefronts per
// SIMD, and these wait for LDS and for one another at each step (walking the lists and staging alone take 184 us).  few_kernel, 32
// sequences with 16 blocks each of 32 / 8 heads of 128: 27.6 us, 4.9 TB/s of keys and values, the rate of a large copy; with less to read
// (1 sequence, 8 heads of 64: 10 us) the chain list, keys, softmax, joining.
#include <algorithm>
#include <type_traits>

#include "fg_block.h"

namespace fg {
namespace block {

namespace {

constexpr int kMergeStride = 36;       // floats between rows of the joining buffer (32 and 4 of padding)

// ---- few queries ------------------------------------------------------------------------------------------

// What gradients start from: a row's scores are relative to the first number, their powers' sum is 2 to the second.  In one number a reference
// beyond 2^24, of a row that sees only masked keys, would take the sum away.
__device__ __forceinline__ float2 log_sum(float reference, float sum) {
    return sum == 0.f ? make_float2(__builtin_inff(), 0.f) : make_float2(reference, __builtin_amdgcn_logf(sum));
}

// How far below the largest score a row's reference stands, in base 2: float16 holds powers from 2^-14 on in full, and a long row's output may be
// that of many small ones.  (They stay below 2^15: many_kernel's reference follows the maximum by up to 2^8.)
template <typename T> constexpr float kBelow = std::is_same<T, _Float16>::value ? 7.f : 0.f;

template <typename T, int D> constexpr size_t few_stage_bytes() {
    const size_t values = (size_t)kWaves * kUnit * (D + kPad) * sizeof(T), merge = (size_t)kWaves * 16 * kMergeStride * sizeof(float);
    return values > merge ? values : merge;
}

struct Results { void *out, *rest; float2 *lse; float *part; float2 *part_stats; };

struct FewShared {
    List<1, 1024> list;
    float2 stats[kWaves][16], joined[16];
};

// One tile of 16 rows, or one of `splits` shares of its list.  CAREFUL: with values that are not finite kept apart from the start.
template <typename T, int D, bool CAREFUL>
__device__ __forceinline__ void few_rows(const Problem &p, const Results &r, FewShared &shared, unsigned char *dynamic, const Buckets &buckets, int b, int h,
                                         int tile, int split, int splits) {
    constexpr int DC = D / 32, DT = D / 16, S = D + kPad;
    constexpr int EPC = 16 / sizeof(T), CPR = D / EPC, RPL = 64 / CPR, NV = kUnit / RPL;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, c = lane & 15;
    const int k_len = key_count(p, b), q_len = query_count(p, b), offset = k_len - q_len;
    const int tpt = tile_tokens(p.group), t0 = tile * tpt;
    const int tc = c / p.group, mine = c - tc * p.group, head = h * p.group + mine;        // this lane's token within the tile, and its head
    const bool used = tc < tpt;

    T *stage = reinterpret_cast<T *>(dynamic) + wave * kUnit * S;
    const bool there = used && t0 + tc < q_len;
    // last key that the lane's row may see (columns without a row see everything, so that they do not keep the tile from skipping its
    // masks; nothing is written of them)
    const int limit = there ? (p.causal ? min(offset + t0 + tc, k_len - 1) : k_len - 1) : used ? -1 : k_len - 1;
    V8<T> qf[DC];
    const T *src = static_cast<const T *>(p.q) + b * p.qs.batch + (int64_t)(t0 + tc) * p.qs.row + head * p.qs.head + 8 * g;
#pragma unroll
    for (int dc = 0; dc < DC; ++dc) qf[dc] = there ? load8(src + dc * 32) : zero8<T>();
    const int last_key = p.causal ? min(k_len - 1, offset + min(t0 + tpt, q_len) - 1) : k_len - 1;
    const T *kbase = static_cast<const T *>(p.k) + b * p.ks.batch + h * p.ks.head + 8 * g;
    const T *vbase = static_cast<const T *>(p.v) + b * p.vs.batch + h * p.vs.head + (lane % CPR) * EPC;
    const int sub_shift = p.block_shift - 5;
    auto &list = shared.list;

    f32x4 o[DT];
    float m, l;
    auto sweep = [&](auto careful) {
        m = -__builtin_inff(); l = 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int first = 0; first < p.blocks; first += list.kWidth) {
            const int units = build_list(list, p, b, h, t0, q_len, k_len, first, min(list.kWidth, p.blocks - first)) << sub_shift;
            auto first_key = [&](int u) {
                return __builtin_amdgcn_readfirstlane(((first + list.id[u >> sub_shift]) << p.block_shift) + ((u & ((1 << sub_shift) - 1)) << 5));
            };
            // the next unit, from u on, that holds a key anyone may see
            auto find = [&](int u) {
                while (u < units && first_key(u) > last_key) u += kWaves * splits;
                return u;
            };
            V8<T> kf[2][DC];
            u32x4 vr[NV];
            int key0 = 0;
            unsigned who = 0;
            auto fetch = [&](int u) {
                key0 = first_key(u);
                who = (unsigned)list.bits[u >> sub_shift][0];
                // rows behind the last key read it again: what a padded cache holds there is never touched
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int dc = 0; dc < DC; ++dc) kf[kt][dc] = load8(kbase + (int64_t)min(key0 + kt * 16 + c, k_len - 1) * p.ks.row + dc * 32);
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    vr[i] = *reinterpret_cast<const u32x4 *>(vbase + (int64_t)min(key0 + i * RPL + lane / CPR, k_len - 1) * p.vs.row);
            };
            int u = find(wave + kWaves * split);
            if (u < units) fetch(u);
            while (u < units) {
                const int now = key0;
                const int last = !used || (who >> tc) & 1 ? limit : -1;      // keys that the lane's row sees: now + 16 kt + 4 g + i <= last
                wave_lds_sync();
#pragma unroll
                for (int i = 0; i < NV; ++i) *reinterpret_cast<u32x4 *>(stage + (i * RPL + lane / CPR) * S + (lane % CPR) * EPC) = vr[i];
                wave_lds_sync();
                f32x4 s[2];
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) {
                    s[kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int dc = 0; dc < DC; ++dc) s[kt] = mma(kf[kt][dc], qf[dc], s[kt]);
                }
                u = find(u + kWaves * splits);
                if (u < units) fetch(u);

                // z = s factor; powers are taken of z - reference in one operation, unrounded between, as many_kernel and the gradients take them
                const float factor = p.n_buckets ? 1.f : p.scale2;
                if (p.n_buckets) {
                    const int pos = offset + t0, near = buckets.at(pos - now - (kUnit - 1)), far = buckets.at(pos + tpt - 1 - now);
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            s[kt][i] = s[kt][i] * p.scale2 + buckets.value(near == far ? near : buckets.at(pos + tc - (now + 16 * kt + 4 * g + i)), mine);
                }
                f32x4 z[2] = {s[0] * factor, s[1] * factor};
                unsigned seen = 0xff;
                if (!__all(now + kUnit - 1 <= last)) {
                    seen = 0;
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const bool ok = now + 16 * kt + 4 * g + i <= last;
                            z[kt][i] = ok ? z[kt][i] : -__builtin_inff();
                            seen |= (unsigned)ok << (4 * kt + i);
                        }
                }
                float top = fmaxf(fmaxf(fmaxf(z[0][0], z[0][1]), fmaxf(z[0][2], z[0][3])), fmaxf(fmaxf(z[1][0], z[1][1]), fmaxf(z[1][2], z[1][3])));
                top = fmaxf(m, rows_max(top) - kBelow<T>);
                const float ref = top == -__builtin_inff() ? 0.f : top;       // nothing above -inf so far: every power below is 0
                if (__any(top != m)) {
                    const float shrink = __builtin_amdgcn_exp2f(m - ref);
                    l *= shrink;
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) o[dt] *= shrink;
                    m = top;
                }
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        s[kt][i] = z[kt][i] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][i], factor, -ref));
                l += ((s[0][0] + s[0][1]) + (s[0][2] + s[0][3])) + ((s[1][0] + s[1][1]) + (s[1][2] + s[1][3]));
                // the powers are rounded to the operands' type for the product with V, half a step each; their sum is not.  What the rounding
                // took follows in a second product, with gradients or without: it takes no time that shows here.
                V8<T> pf, pl;
                block::split<T>(s[0], s[1], &pf, &pl);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    const V8<T> vf = transposed<T, D>(stage, dt * 16, lane);
                    if constexpr (decltype(careful)::value) o[dt] = mma_masked<T>(vf, pf, pl, seen, o[dt]);
                    else o[dt] = mma(vf, pf, o[dt]);
                }
                if (sizeof(T) == 2 && !decltype(careful)::value)
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) o[dt] = mma(transposed<T, D>(stage, dt * 16, lane), pl, o[dt]);
            }
        }
    };
    if constexpr (CAREFUL) {
        sweep(std::true_type{});
    } else {
        sweep(std::false_type{});
        bool odd = false;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) odd |= not_finite(o[dt]);
        if (__syncthreads_or(odd)) sweep(std::true_type{});
    }

    // the four wavefronts' sums, joined a strip of 32 columns at a time
    l = rows_sum(l);
    __syncthreads();                   // the joining buffer of the tile before has been read
    if (g == 0) shared.stats[wave][c] = make_float2(m, l);
    __syncthreads();
    float top = -__builtin_inff(), total = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, shared.stats[w][c].x);
    const float ref = top == -__builtin_inff() ? 0.f : top;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) total += shared.stats[w][c].y * __builtin_amdgcn_exp2f(shared.stats[w][c].x - ref);
    const float share = __builtin_amdgcn_exp2f(m - ref);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] *= share;
    if (wave == 0 && g == 0) shared.joined[c] = make_float2(top, total);
    float *merge = reinterpret_cast<float *>(dynamic);
    const int64_t all_rows = (int64_t)p.batch * p.queries * p.heads;
#pragma unroll
    for (int strip = 0; strip < DC; ++strip) {
        __syncthreads();               // the values' staging, or the strip before, has been read
#pragma unroll
        for (int j = 0; j < 2; ++j) *reinterpret_cast<f32x4 *>(merge + (wave * 16 + c) * kMergeStride + 16 * j + 4 * g) = o[2 * strip + j];
        __syncthreads();
        const int row = tid >> 3, col = (tid & 7) * 4, rt = row / p.group, t = t0 + rt;
        if (tid < 16 * 8 && rt < tpt && t < p.queries) {
            f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < kWaves; ++w) sum += *reinterpret_cast<const f32x4 *>(merge + (w * 16 + row) * kMergeStride + col);
            const int64_t at = ((int64_t)b * p.queries + t) * p.heads + h * p.group + (row - rt * p.group);
            const float2 st = shared.joined[row];
            if (splits == 1) {
                const float inv = st.y == 0.f ? 0.f : 1.f / st.y;
                store_row<T>(static_cast<T *>(r.out), static_cast<T *>(r.rest), at * D + strip * 32 + col, sum * inv);
                if (strip == 0 && col == 0 && r.lse) r.lse[at] = log_sum(st.x, st.y);
            } else {
                *reinterpret_cast<f32x4 *>(r.part + (split * all_rows + at) * D + strip * 32 + col) = sum;
                if (strip == 0 && col == 0) r.part_stats[split * all_rows + at] = st;
            }
        }
    }
}

template <typename T, int D>
__global__ __launch_bounds__(kThreads) void few_kernel(const Problem p, const Results r, int n_tiles, int splits) {
    __shared__ FewShared shared;
    extern __shared__ __align__(16) unsigned char dynamic[];
    const int unit = xcd_contiguous_block(), pair = unit / (n_tiles * splits), rest = unit - pair * n_tiles * splits, tile = rest / splits;
    const int b = pair / p.kv_heads, h = pair - b * p.kv_heads;
    Buckets buckets;
    if (p.n_buckets) buckets = load_buckets<T>(p, h, dynamic + few_stage_bytes<T, D>());
    few_rows<T, D, false>(p, r, shared, dynamic, buckets, b, h, tile, rest - tile * splits, splits);
}

// ---- many queries -----------------------------------------------------------------------------------------

constexpr int kStep = 64;              // keys in LDS
constexpr int kListed = 256;           // blocks listed at a time

template <typename T, int D> struct Steps {
    static constexpr int kKeyStride = D + 16 / sizeof(T), kValueStride = D + kPad;
    static constexpr size_t kStepBytes = (size_t)kStep * (kKeyStride + kValueStride) * sizeof(T);
    static constexpr int kBuffers = kStepBytes <= 40 * 1024 ? 2 : 1;      // two workgroups' worth fits a CU's LDS
    static constexpr size_t kBytes = kBuffers * kStepBytes;
};

// RT tiles of 16 rows per wavefront.  flags[workgroup]: whether a result was not finite (see redo_kernel).
// EXACT: what the powers' rounding took goes into a second product with V.  Gradients start from <dO, O>, which a row's dS takes away from
// numbers of its own size: with rounded powers it would be further off than the gradients' own rounding.  Without gradients the powers' rounding
// is of the size of the output's own, and the second product is left out (8,192 tokens, 32 / 8 heads 372 and 450 us).
template <typename T, int D, int RT, bool BIAS, bool EXACT>
__global__ __launch_bounds__(kThreads, 2) void many_kernel(const Problem p, const Results r, int32_t *flags, int n_groups) {
    constexpr int DC = D / 32, DT = D / 16, TILES = kWaves * RT;
    constexpr int KS = Steps<T, D>::kKeyStride, VS = Steps<T, D>::kValueStride;
    __shared__ List<TILES, kListed> list;
    extern __shared__ __align__(16) unsigned char dynamic[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, c = lane & 15;
    const int unit = xcd_contiguous_block(), pair = unit / n_groups, b = pair / p.kv_heads, h = pair - b * p.kv_heads;
    const int k_len = key_count(p, b), q_len = query_count(p, b), offset = k_len - q_len;
    const int tpt = tile_tokens(p.group), t0 = group_of(p, unit - pair * n_groups, n_groups) * TILES * tpt;
    const int tc = c / p.group, mine = c - tc * p.group, head = h * p.group + mine;
    const bool used = tc < tpt;

    T *tiles = reinterpret_cast<T *>(dynamic);
    constexpr int BUFFERS = Steps<T, D>::kBuffers;
    Buckets buckets;
    if (BIAS) buckets = load_buckets<T>(p, h, dynamic + Steps<T, D>::kBytes);

    // scores are compared before they are scaled: a negative scale turns the queries' signs instead
    const float factor = BIAS ? 1.f : fabsf(p.scale2);
    V8<T> qf[RT][DC];
    int limit[RT];                     // last key that the lane's row may see; columns without a row see everything, nothing is written of them
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int t = t0 + (wave * RT + rt) * tpt + tc;
        const bool there = used && t < q_len;
        limit[rt] = there ? (p.causal ? min(offset + t, k_len - 1) : k_len - 1) : used ? -1 : k_len - 1;
        const T *src = static_cast<const T *>(p.q) + b * p.qs.batch + (int64_t)t * p.qs.row + head * p.qs.head + 8 * g;
#pragma unroll
        for (int dc = 0; dc < DC; ++dc) qf[rt][dc] = there ? load8(src + dc * 32) : zero8<T>();
        if (!BIAS && p.scale2 < 0.f)
#pragma unroll
            for (int dc = 0; dc < DC; ++dc) qf[rt][dc] = -qf[rt][dc];
    }
    const int last_key = p.causal ? min(k_len - 1, offset + min(t0 + TILES * tpt, q_len) - 1) : k_len - 1;
    const T *kbase = static_cast<const T *>(p.k) + b * p.ks.batch + h * p.ks.head;
    const T *vbase = static_cast<const T *>(p.v) + b * p.vs.batch + h * p.vs.head;
    const int sub_shift = p.block_shift - 5;

    // The sum that divides the output is that of the rounded powers, which are the weights of the product (a product with ones makes it):
    // a row that one key dominates keeps that key's value to the last bit.
    f32x4 o[RT][DT], total[RT];
    float m[RT], l[RT];
    V8<T> ones;
#pragma unroll
    for (int i = 0; i < 8; ++i) ones[i] = (T)1.f;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -__builtin_inff(); l[rt] = 0.f;
        total[rt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[rt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (int first = 0; first < p.blocks; first += kListed) {
        const int units = build_list(list, p, b, h, t0, q_len, k_len, first, min(kListed, p.blocks - first)) << sub_shift;
        // a step is two units of 32 keys, of one block or (blocks of 32) of two
        auto first_key = [&](int u) {
            return __builtin_amdgcn_readfirstlane(((first + list.id[u >> sub_shift]) << p.block_shift) + ((u & ((1 << sub_shift) - 1)) << 5));
        };
        Stage<T, D> ks, vs;
        // ids of the step after the next, and the next step's tokens, are on their way while a step is worked on
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
            if (!(sel[0] | sel[1])) continue;        // none of the wavefront's tokens selected these blocks
            V8<T> kf[2][DC];
            auto read_keys = [&](int x) {
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int dc = 0; dc < DC; ++dc) kf[kt][dc] = load8(keys + (x * kUnit + kt * 16 + c) * KS + dc * 32 + 8 * g);
            };
            read_keys(sel[0] ? 0 : 1);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                if (!sel[x]) continue;
                f32x4 s[RT][2];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt) s[rt][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int dc = 0; dc < DC; ++dc)
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt) s[rt][kt] = mma(kf[kt][dc], qf[rt][dc], s[rt][kt]);
                // the next keys and the first half of the values are read while the powers are taken
                if (x == 0 && sel[1]) read_keys(1);
                V8<T> vf[DT / 2];
                auto read_values = [&](int half) {
#pragma unroll
                    for (int i = 0; i < DT / 2; ++i) vf[i] = transposed<T, D>(values + x * kUnit * VS, (half * (DT / 2) + i) * 16, lane);
                };
                read_values(0);
                __builtin_amdgcn_sched_barrier(0);
                bool mine_too[RT], edge = false;     // whether the lane's row selected the block
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    mine_too[rt] = !used || (sel[x] >> (16 * rt + tc)) & 1;
                    edge |= mine_too[rt] && key0[x] + kUnit - 1 > limit[rt];
                }
                if (BIAS) {
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        const int pos = offset + t0 + (wave * RT + rt) * tpt;
                        const int near = buckets.at(pos - key0[x] - (kUnit - 1)), far = buckets.at(pos + tpt - 1 - key0[x]);
                        const float y = near == far ? buckets.value(near, mine) : 0.f;
#pragma unroll
                        for (int i = 0; i < 4; ++i) { s[rt][0][i] = s[rt][0][i] * p.scale2 + y; s[rt][1][i] = s[rt][1][i] * p.scale2 + y; }
                        if (near != far)
#pragma unroll
                            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                                for (int i = 0; i < 4; ++i) s[rt][kt][i] += buckets.value(buckets.at(pos + tc - (key0[x] + 16 * kt + 4 * g + i)), mine);
                    }
                }
                // a row that did not select the block has its powers taken from +inf: 0, whatever finite scores it has there.  Only keys
                // behind a row that did are masked one by one.
                if (__any(edge)) {
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        const int last = (mine_too[rt] ? limit[rt] : -1) - key0[x] - 4 * g;
#pragma unroll
                        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                            for (int i = 0; i < 4; ++i) s[rt][kt][i] = 16 * kt + i <= last ? s[rt][kt][i] : -__builtin_inff();
                    }
                }
                float high[RT];
                bool moved = false;
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    const float most = largest(s[rt][0], s[rt][1]);
                    high[rt] = largest_of_rows(mine_too[rt] ? most : -__builtin_inff()) * factor - kBelow<T>;
                    moved |= high[rt] > m[rt] + 8.f;
                }
                // sums are kept relative to a reference that follows the maximum when it has moved by more than 2^8
                if (__any(moved)) {
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        const float up = fmaxf(m[rt], high[rt]), from = up == -__builtin_inff() ? 0.f : up;
                        const float shrink = __builtin_amdgcn_exp2f(m[rt] - from);
                        l[rt] *= shrink;
                        total[rt] *= shrink;
#pragma unroll
                        for (int dt = 0; dt < DT; ++dt) o[rt][dt] *= shrink;
                        m[rt] = up;
                    }
                }
                V8<T> pf[RT], pl[RT];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    float from = m[rt] == -__builtin_inff() ? 0.f : m[rt];
                    from = mine_too[rt] ? from : __builtin_inff();
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[rt][kt][i] = __builtin_amdgcn_exp2f(s[rt][kt][i] * factor - from);
                    // rounded to the operands' type for the product with V, half a step each
                    if (EXACT) split<T>(s[rt][0], s[rt][1], &pf[rt], &pl[rt]);
                    else pf[rt] = pack<T>(s[rt][0], s[rt][1]);
                }
                if (r.lse)
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        const f32x4 a = s[rt][0] + s[rt][1];
                        l[rt] += (a[0] + a[1]) + (a[2] + a[3]);
                    }
#pragma unroll
                for (int half = 0; half < 2; ++half) {
#pragma unroll
                    for (int i = 0; i < DT / 2; ++i)
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt) {
                            o[rt][half * (DT / 2) + i] = mma(vf[i], pf[rt], o[rt][half * (DT / 2) + i]);
                            if (EXACT) o[rt][half * (DT / 2) + i] = mma(vf[i], pl[rt], o[rt][half * (DT / 2) + i]);
                        }
                    if (half == 0) read_values(1);
                }
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    total[rt] = mma(ones, pf[rt], total[rt]);
                    if (EXACT) total[rt] = mma(ones, pl[rt], total[rt]);
                }
            }
        }
    }
    bool odd = false;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const float inv = total[rt][0] == 0.f ? 0.f : 1.f / total[rt][0], sum = rows_sum(l[rt]);
        const int t = t0 + (wave * RT + rt) * tpt + tc;
        const int64_t at = ((int64_t)b * p.queries + t) * p.heads + head;
        const bool write = used && t < p.queries;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            odd |= not_finite(o[rt][dt]);
            if (write) store_row<T>(static_cast<T *>(r.out), static_cast<T *>(r.rest), at * D + dt * 16 + 4 * g, o[rt][dt] * inv);
        }
        if (write && g == 0 && r.lse) r.lse[at] = log_sum(m[rt], sum);
    }
    odd = __syncthreads_or(odd);
    if (tid == 0) flags[unit] = odd;
}

// The tiles of many_kernel's workgroups with a result that was not finite, again.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void redo_kernel(const Problem p, const Results r, const int32_t *flags, int n_groups, int tiles) {
    __shared__ FewShared shared;
    extern __shared__ __align__(16) unsigned char dynamic[];
    const int unit = xcd_contiguous_block();
    if (!flags[unit]) return;
    const int pair = unit / n_groups, b = pair / p.kv_heads, h = pair - b * p.kv_heads, first = group_of(p, unit - pair * n_groups, n_groups) * tiles;
    Buckets buckets;
    if (p.n_buckets) buckets = load_buckets<T>(p, h, dynamic + few_stage_bytes<T, D>());
    for (int i = 0; i < tiles; ++i) few_rows<T, D, true>(p, r, shared, dynamic, buckets, b, h, first + i, 0, 1);
}

// Joins the sums of several workgroups per row: four columns a thread.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void join_kernel(const float *part, const float2 *part_stats, T *out, T *remainder, float2 *lse, int64_t rows, int splits) {
    const int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x, row = e / (D / 4);
    const int col = (int)(e - row * (D / 4)) * 4;
    if (row >= rows) return;
    float top = -__builtin_inff(), total = 0.f;
    for (int s = 0; s < splits; ++s) top = fmaxf(top, part_stats[s * rows + row].x);
    const float ref = top == -__builtin_inff() ? 0.f : top;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < splits; ++s) {
        const float2 st = part_stats[s * rows + row];
        const float share = __builtin_amdgcn_exp2f(st.x - ref);
        total += st.y * share;
        sum += *reinterpret_cast<const f32x4 *>(part + (s * rows + row) * D + col) * share;
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    store_row<T>(out, remainder, row * D + col, sum * inv);
    if (col == 0 && lse) lse[row] = log_sum(top, total);
}

// Which kernel takes a call, and how its work is cut.  many_kernel wants its workgroups' tiles at least half full and 256 workgroups (a CU each).
// Both sides, few_kernel / many_kernel, heads of 128 in bfloat16, 16 blocks of 64.  One sequence of 32 / 8 heads: 256 tokens (64 workgroups)
// 19 / 18 us, 512 40 / 26, 1,024 (256 workgroups) 98 / 42, 2,048 257 / 71.  32 sequences of 8 / 8 heads over 2,048 keys: 16 tokens (an eighth
// of a workgroup's rows) 49 / 67, 32 61 / 70, 48 86 / 73, 64 112 / 74, 128 213 / 80.  In 32 bits, heads of 64, 8 blocks of 32, two sequences of 8
// heads: 1,024 tokens (256 workgroups) 41 / 53, 2,048 82 / 89.  So the cut comes late for long lists in 16 bits and early for short ones in 32.
// few_kernel's workgroups take about 8 us and 0.35 us for each unit of a wavefront, and joining several costs 6 us with its launch: a list
// is dealt out to several workgroups where a wavefront would have more than eight units of it, then down to four.
struct Shape { bool many; int n_tiles, splits; };
template <int RT> Shape shape_of(const Problem &p) {
    const int tpt = tile_tokens(p.group);
    const int64_t pairs = (int64_t)p.batch * p.kv_heads;
    auto tiles = [&](int n) { return (p.queries + n * tpt - 1) / (n * tpt); };
    Shape s{true, tiles(kWaves * RT), 1};
    if (pairs * s.n_tiles >= 256 && 2 * p.queries >= kWaves * RT * tpt) return s;
    s = Shape{false, tiles(1), 1};
    const int64_t groups = std::max<int64_t>(pairs * s.n_tiles, 1);
    const int64_t named = std::min<int64_t>((int64_t)p.topk * std::min(tpt, p.queries), p.blocks);
    const int64_t units = named << (p.block_shift - 5);            // of a list at most
    if (units > 8 * kWaves) s.splits = (int)std::max<int64_t>(1, std::min<int64_t>((512 + groups - 1) / groups, units / (4 * kWaves)));
    return s;
}

size_t round_up(size_t n) { return (n + 255) & ~(size_t)255; }

template <typename T, int D>
int launch(const Problem &p, const fg_block_attention_args *a, void *workspace, size_t bytes, size_t *need, hipStream_t stream) {
    constexpr int RT = sizeof(T) == 4 ? 1 : 2;
    const Shape s = shape_of<RT>(p);
    const size_t rows = (size_t)p.batch * p.queries * p.heads;
    const int64_t grid = (int64_t)p.batch * p.kv_heads * s.n_tiles * s.splits;
    if (grid >= (1ll << 31)) return fail(FG_ERR_SHAPE, "block attention: %lld workgroups do not fit a launch", (long long)grid);
    const size_t flags = s.many ? round_up((size_t)grid * sizeof(int32_t)) : 0;
    const size_t sums = s.splits > 1 ? round_up(rows * s.splits * D * sizeof(float)) : 0, stats = s.splits > 1 ? round_up(rows * s.splits * sizeof(float2)) : 0;
    if (need) { *need = flags + sums + stats; return FG_OK; }
    if (bytes < flags + sums + stats || (flags + sums && !workspace))
        return fail(FG_ERR_ARG, "block attention: a workspace of %zu bytes, %zu needed (fg_block_attention_workspace)", bytes, flags + sums + stats);
    unsigned char *w = static_cast<unsigned char *>(workspace);
    const Results r{a->out, a->rest, reinterpret_cast<float2 *>(a->lse), reinterpret_cast<float *>(w), reinterpret_cast<float2 *>(w + sums)};
    const size_t bias = buckets_bytes(p.n_buckets, p.low, p.high, p.group);
    const dim3 blocks((unsigned)grid), threads(kThreads);
    if (s.many) {
        int32_t *marks = reinterpret_cast<int32_t *>(w);
        auto go = [&](auto exact) {
            constexpr bool EXACT = decltype(exact)::value;
            if (p.n_buckets) many_kernel<T, D, RT, true, EXACT><<<blocks, threads, Steps<T, D>::kBytes + bias, stream>>>(p, r, marks, s.n_tiles);
            else many_kernel<T, D, RT, false, EXACT><<<blocks, threads, Steps<T, D>::kBytes, stream>>>(p, r, marks, s.n_tiles);
        };
        if constexpr (sizeof(T) == 2) {
            if (r.rest) go(std::true_type{});
            else go(std::false_type{});
        } else {
            go(std::false_type{});
        }
        FG_HIP_TRY(hipGetLastError());
        redo_kernel<T, D><<<blocks, threads, few_stage_bytes<T, D>() + bias, stream>>>(p, r, marks, s.n_tiles, kWaves * RT);
    } else {
        few_kernel<T, D><<<blocks, threads, few_stage_bytes<T, D>() + bias, stream>>>(p, r, s.n_tiles, s.splits);
    }
    FG_HIP_TRY(hipGetLastError());
    if (s.splits == 1) return FG_OK;
    const int64_t each = (int64_t)rows * (D / 4);
    join_kernel<T, D><<<dim3((unsigned)((each + kThreads - 1) / kThreads)), threads, 0, stream>>>(
        r.part, r.part_stats, static_cast<T *>(r.out), static_cast<T *>(r.rest), r.lse, (int64_t)rows, s.splits);
    FG_HIP_TRY(hipGetLastError());
    return FG_OK;
}

template <typename T> int launch_d(const Problem &p, const fg_block_attention_args *a, void *workspace, size_t bytes, size_t *need, hipStream_t stream) {
    switch (a->head_len) {
    case 32: return launch<T, 32>(p, a, workspace, bytes, need, stream);
    case 64: return launch<T, 64>(p, a, workspace, bytes, need, stream);
    default: return launch<T, 128>(p, a, workspace, bytes, need, stream);
    }
}

int launch_t(const Problem &p, const fg_block_attention_args *a, void *workspace, size_t bytes, size_t *need, hipStream_t stream) {
    switch (a->type) {
    case FG_TYPE_F32: return launch_d<float>(p, a, workspace, bytes, need, stream);
    case FG_TYPE_F16: return launch_d<_Float16>(p, a, workspace, bytes, need, stream);
    default: return launch_d<__bf16>(p, a, workspace, bytes, need, stream);
    }
}

}  // namespace

int aligned(const char *name, const void *ptr, int bytes, const char *what) {
    return reinterpret_cast<uintptr_t>(ptr) % bytes ? fail(FG_ERR_ARG, "%s: %s has to stand at a multiple of %d bytes", what, name, bytes) : FG_OK;
}

int strides_of(const char *name, const void *ptr, const int64_t *stride, int size, Strides *s, const char *what) {
    const int64_t per = 16 / size;
    if (reinterpret_cast<uintptr_t>(ptr) % 16 || stride[0] % per || stride[1] % per || stride[2] % per)
        return fail(FG_ERR_ARG, "%s: %s and its strides have to be multiples of 16 bytes", what, name);
    *s = Strides{stride[0], stride[1], stride[2]};
    return FG_OK;
}

int problem_of(const fg_block_attention_args *a, Problem *p) {
    if (!a) return fail(FG_ERR_ARG, "block attention: arguments are a null pointer");
    if (a->type != FG_TYPE_F32 && a->type != FG_TYPE_F16 && a->type != FG_TYPE_BF16) return fail(FG_ERR_ARG, "block attention: unknown type %d", a->type);
    if (a->batch < 0 || a->queries < 0 || a->keys < 0 || a->heads < 1 || a->kv_heads < 1 || a->topk < 1)
        return fail(FG_ERR_ARG, "block attention: negative sizes, or no heads or blocks per query");
    if (a->head_len != 32 && a->head_len != 64 && a->head_len != 128) return fail(FG_ERR_SHAPE, "block attention: heads of 32, 64 or 128 elements, got %d", a->head_len);
    if (a->block != 32 && a->block != 64 && a->block != 128 && a->block != 256) return fail(FG_ERR_SHAPE, "block attention: blocks of 32, 64, 128 or 256 keys, got %d", a->block);
    if (a->heads % a->kv_heads || a->heads / a->kv_heads > 16)
        return fail(FG_ERR_SHAPE, "block attention: %d heads over %d key heads: the former have to be 1 to 16 times the latter", a->heads, a->kv_heads);
    // positions, keys and the rows of a list are counted in 32 bits; the arrays behind them are addressed in 64
    if (a->keys > (1 << 30) || a->queries > (1 << 30) || (int64_t)a->topk * 128 > INT32_MAX / a->kv_heads)
        return fail(FG_ERR_SHAPE, "block attention: more than 2^30 keys or queries, or too long a list");
    if (a->n_buckets < 0 || a->n_buckets > 64) return fail(FG_ERR_SHAPE, "block attention: %d buckets: 1 to 64, or 0 for no bias", a->n_buckets);
    *p = Problem{};
    p->low = p->high = 0;
    for (int i = 0; i + 1 < a->n_buckets; ++i) {
        p->bounds[i] = a->bounds[i];
        if (i && a->bounds[i] <= a->bounds[i - 1]) return fail(FG_ERR_ARG, "block attention: the buckets' bounds have to ascend");
    }
    if (a->n_buckets > 1) {
        if (a->bounds[0] < -(1 << 30) || a->bounds[a->n_buckets - 2] > (1 << 30) || a->bounds[a->n_buckets - 2] - a->bounds[0] >= kSpan - 1)
            return fail(FG_ERR_SHAPE, "block attention: the first and the last bound are %d distances apart at most", kSpan - 2);
        p->low = a->bounds[0] - 1;
        p->high = a->bounds[a->n_buckets - 2];
    }
    const int size = a->type == FG_TYPE_F32 ? 4 : 2;
    int rc;
    if ((rc = strides_of("q", a->q, a->q_strides, size, &p->qs)) || (rc = strides_of("k", a->k, a->k_strides, size, &p->ks)) ||
        (rc = strides_of("v", a->v, a->v_strides, size, &p->vs)) || (rc = aligned("out", a->out, 16)) || (rc = aligned("rest", a->rest, 16)) ||
        (rc = aligned("lse", a->lse, 8)) || (rc = aligned("blocks", a->blocks, 4)) || (rc = aligned("lengths", a->lengths, 4)) ||
        (rc = aligned("q_lengths", a->q_lengths, 4)) || (rc = aligned("bias", a->bias, size))) return rc;
    p->batch = a->batch; p->queries = a->queries; p->keys = a->keys; p->heads = a->heads; p->kv_heads = a->kv_heads; p->group = a->heads / a->kv_heads;
    p->block_shift = a->block == 32 ? 5 : a->block == 64 ? 6 : a->block == 128 ? 7 : 8;
    p->blocks = (a->keys + a->block - 1) / a->block;
    p->topk = a->topk; p->causal = a->causal != 0; p->scale = a->scale; p->scale2 = a->scale * kLog2e;
    p->q = a->q; p->k = a->k; p->v = a->v; p->bias = a->bias; p->list = a->blocks; p->lengths = a->lengths; p->q_lengths = a->q_lengths;
    p->n_buckets = a->n_buckets;
    return FG_OK;
}
}  // namespace block
}  // namespace fg

extern "C" int64_t fg_block_attention_workspace(const fg_block_attention_args *args) {
    fg::block::Problem p;
    if (int rc = fg::block::problem_of(args, &p)) return rc;
    size_t need = 0;
    const int rc = fg::block::launch_t(p, args, nullptr, 0, &need, nullptr);
    return rc ? rc : (int64_t)need;
}

extern "C" int fg_block_attention(const fg_block_attention_args *args, void *workspace, size_t workspace_bytes, void *stream) {
    fg::block::Problem p;
    if (int rc = fg::block::problem_of(args, &p)) return rc;
    if ((int64_t)p.batch * p.queries == 0) return FG_OK;
    if (!p.q || !p.list || !args->out || (p.keys && (!p.k || !p.v)) || (p.n_buckets && !p.bias)) return fg::fail(FG_ERR_ARG, "block attention: null pointer");
    if (int rc = fg::block::aligned("the workspace", workspace, 16)) return rc;
    return fg::block::launch_t(p, args, workspace, workspace_bytes, nullptr, static_cast<hipStream_t>(stream));
}
