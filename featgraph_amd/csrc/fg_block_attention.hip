// Softmax attention over the blocks of keys that every query selected, forward:
//   out[i, h] = sum_j p_ij V[j, g],  p_i = softmax over the visible keys j of  scale <Q[i, h], K[j, g]> + bias[bucket(pos_i - j), h]
// with g = h / group, pos_i = k_len - q_len + i, and j visible to i where floor(j / block) is in i's list for g, j < k_len and (causal) j <= pos_i.
// No visible key: 0.
//
// One workgroup takes the tokens of RT tiles of 16 rows (16 / group tokens each, all heads of the group) and walks the blocks that any of
// them selected; neighbouring tokens share most of theirs, so a block's keys are fetched once for all of them.  Its four wavefronts
// take 32 keys each in turn and keep a softmax (maximum, sum) and an output of their own, joined at the end: no barrier inside the
// walk.  Keys go from memory into registers as the left operand of (keys x queries); values through a wavefront's own LDS, from which they
// are read with keys along the registers.  A tile none of whose tokens selected a block skips it.
// Where there are few queries, the list is dealt out over several workgroups too, and a second kernel joins their sums.
// Values that are not finite reach the rows that see them and no others: a result that is not finite is computed again
// with such places apart (mma_masked).
#include <algorithm>
#include <type_traits>

#include "fg_block.h"

namespace fg {
namespace block {

namespace {

constexpr int kMergeStride = 36;       // floats between rows of the joining buffer (32 and 4 of padding)

template <typename T, int D, int RT> constexpr size_t stage_bytes() {
    const size_t values = (size_t)kWaves * kUnit * (D + kPad) * sizeof(T), merge = (size_t)kWaves * RT * 16 * kMergeStride * sizeof(float);
    return values > merge ? values : merge;
}

template <typename T, int D, int RT>
__global__ __launch_bounds__(kThreads) void block_attention_kernel(const Problem p, T *out, T *remainder, float *lse, float *part, float2 *part_stats,
                                                                   int n_tiles, int splits) {
    constexpr int DC = D / 32, DT = D / 16, S = D + kPad;
    constexpr int EPC = 16 / sizeof(T), CPR = D / EPC, RPL = 64 / CPR, NV = kUnit / RPL;
    __shared__ List list;
    __shared__ float2 stats[kWaves][RT * 16];
    __shared__ float2 joined[RT * 16];
    extern __shared__ __align__(16) unsigned char dynamic[];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, c = lane & 15;
    const int unit = xcd_contiguous_block();
    const int pair = unit / (n_tiles * splits), rest = unit - pair * n_tiles * splits;
    const int tile = rest / splits, split = rest - tile * splits;
    const int b = pair / p.kv_heads, h = pair - b * p.kv_heads;
    const int k_len = key_count(p, b), q_len = query_count(p, b), offset = k_len - q_len;
    const int tpt = tile_tokens(p.group), t0 = tile * RT * tpt, nt = RT * tpt;
    const int tc = c / p.group, head = h * p.group + (c - tc * p.group);        // this lane's token within a tile, and its head
    const bool used = tc < tpt;

    T *stage = reinterpret_cast<T *>(dynamic) + wave * kUnit * S;
    Buckets buckets;
    if (p.n_buckets) buckets = load_buckets<T>(p, h, dynamic + stage_bytes<T, D, RT>());

    V8<T> qf[RT][DC];
    int limit[RT];                     // last key that the lane's row may see
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int t = t0 + rt * tpt + tc;
        const bool there = used && t < q_len;
        // (columns without a row see everything, so that they do not keep a tile from skipping its masks; nothing is written of them)
        limit[rt] = there ? (p.causal ? min(offset + t, k_len - 1) : k_len - 1) : used ? -1 : k_len - 1;
        const T *src = static_cast<const T *>(p.q) + b * p.qs.batch + (int64_t)t * p.qs.row + head * p.qs.head + 8 * g;
#pragma unroll
        for (int dc = 0; dc < DC; ++dc) qf[rt][dc] = there ? load8(src + dc * 32) : zero8<T>();
    }
    const int last_key = p.causal ? min(k_len - 1, offset + min(t0 + nt, q_len) - 1) : k_len - 1;
    const T *kbase = static_cast<const T *>(p.k) + b * p.ks.batch + h * p.ks.head + 8 * g;
    const T *vbase = static_cast<const T *>(p.v) + b * p.vs.batch + h * p.vs.head + (lane % CPR) * EPC;
    const int sub_shift = p.block_shift - 5;

    f32x4 o[RT][DT];
    float m[RT], l[RT];
    auto sweep = [&](auto careful) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            m[rt] = -__builtin_inff(); l[rt] = 0.f;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[rt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        for (int first = 0; first < p.blocks; first += kWindow) {
            const int units = build_list(list, p, b, h, t0, nt, q_len, k_len, first, min(kWindow, p.blocks - first)) << sub_shift;
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
            unsigned long long bits = 0;
            auto fetch = [&](int u) {
                key0 = first_key(u);
                bits = uniform64(list.bits[u >> sub_shift]);
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
                const unsigned long long who = bits;
                wave_lds_sync();
#pragma unroll
                for (int i = 0; i < NV; ++i) *reinterpret_cast<u32x4 *>(stage + (i * RPL + lane / CPR) * S + (lane % CPR) * EPC) = vr[i];
                wave_lds_sync();
                f32x4 s[RT][2];
                unsigned active = 0;
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    if (!((who >> (rt * tpt)) & ((1ull << tpt) - 1))) continue;
                    active |= 1u << rt;
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt) {
                        s[rt][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int dc = 0; dc < DC; ++dc) s[rt][kt] = mma(kf[kt][dc], qf[rt][dc], s[rt][kt]);
                    }
                }
                u = find(u + kWaves * splits);
                if (u < units) fetch(u);

                V8<T> pf[RT];
                unsigned seen[RT];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    if (!(active & (1u << rt))) continue;
                    // keys that the lane's row sees: now + 16 kt + 4 g + i <= last
                    const int last = !used || (who >> (rt * tpt + tc)) & 1 ? limit[rt] : -1;
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[rt][kt][i] *= p.scale2;
                    if (p.n_buckets) {
                        const int pos = offset + t0 + rt * tpt, near = buckets.at(pos - now - (kUnit - 1)), far = buckets.at(pos + tpt - 1 - now);
                        const int mine = c - tc * p.group;
                        if (near == far) {
                            const float x = buckets.value(near, mine);
#pragma unroll
                            for (int i = 0; i < 4; ++i) { s[rt][0][i] += x; s[rt][1][i] += x; }
                        } else {
#pragma unroll
                            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                                for (int i = 0; i < 4; ++i) s[rt][kt][i] += buckets.value(buckets.at(pos + tc - (now + 16 * kt + 4 * g + i)), mine);
                        }
                    }
                    unsigned mask = 0xff;
                    if (!__all(now + kUnit - 1 <= last)) {
                        mask = 0;
#pragma unroll
                        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const bool ok = now + 16 * kt + 4 * g + i <= last;
                                s[rt][kt][i] = ok ? s[rt][kt][i] : -__builtin_inff();
                                mask |= (unsigned)ok << (4 * kt + i);
                            }
                    }
                    seen[rt] = mask;
                    const f32x4 a = s[rt][0], e = s[rt][1];
                    float top = fmaxf(fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3])), fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3])));
                    top = fmaxf(m[rt], rows_max(top));
                    const float ref = top == -__builtin_inff() ? 0.f : top;       // nothing above -inf so far: every power below is 0
                    if (__any(top != m[rt])) {
                        const float shrink = __builtin_amdgcn_exp2f(m[rt] - ref);
                        l[rt] *= shrink;
#pragma unroll
                        for (int dt = 0; dt < DT; ++dt) o[rt][dt] *= shrink;
                        m[rt] = top;
                    }
                    f32x4 x, y;
#pragma unroll
                    for (int i = 0; i < 4; ++i) { x[i] = __builtin_amdgcn_exp2f(a[i] - ref); y[i] = __builtin_amdgcn_exp2f(e[i] - ref); }
                    l[rt] += ((x[0] + x[1]) + (x[2] + x[3])) + ((y[0] + y[1]) + (y[2] + y[3]));
                    // the powers are rounded to the operands' type for the product with V, half a step each; their sum is not
                    pf[rt] = pack<T>(x, y);
                }
                if (!careful && active == (1u << RT) - 1) {
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) {
                        const V8<T> vf = transposed<T, D>(stage, dt * 16, lane);
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt) o[rt][dt] = mma(vf, pf[rt], o[rt][dt]);
                    }
                } else {
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        if (!(active & (1u << rt))) continue;
#pragma unroll
                        for (int dt = 0; dt < DT; ++dt) {
                            const V8<T> vf = transposed<T, D>(stage, dt * 16, lane);
                            if constexpr (decltype(careful)::value) o[rt][dt] = mma_masked<T>(vf, pf[rt], seen[rt], o[rt][dt]);
                            else o[rt][dt] = mma(vf, pf[rt], o[rt][dt]);
                        }
                    }
                }
            }
        }
    };
    sweep(std::false_type{});
    bool odd = false;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) odd |= not_finite(o[rt][dt]);
    if (__syncthreads_or(odd)) sweep(std::true_type{});

    // the four wavefronts' sums, joined a strip of 32 columns at a time
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        l[rt] = rows_sum(l[rt]);
        if (g == 0) stats[wave][rt * 16 + c] = make_float2(m[rt], l[rt]);
    }
    __syncthreads();
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        float top = -__builtin_inff(), total = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) top = fmaxf(top, stats[w][rt * 16 + c].x);
        const float ref = top == -__builtin_inff() ? 0.f : top;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) total += stats[w][rt * 16 + c].y * __builtin_amdgcn_exp2f(stats[w][rt * 16 + c].x - ref);
        const float share = __builtin_amdgcn_exp2f(m[rt] - ref);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[rt][dt] *= share;
        if (wave == 0 && g == 0) joined[rt * 16 + c] = make_float2(top, total);
    }
    float *merge = reinterpret_cast<float *>(dynamic);
    const int64_t all_rows = (int64_t)p.batch * p.queries * p.heads;
#pragma unroll
    for (int strip = 0; strip < DC; ++strip) {
        __syncthreads();               // the values' staging, or the strip before, has been read
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                *reinterpret_cast<f32x4 *>(merge + ((wave * RT + rt) * 16 + c) * kMergeStride + 16 * j + 4 * g) = o[rt][2 * strip + j];
        __syncthreads();
        for (int e = tid; e < RT * 16 * 8; e += kThreads) {
            const int row = e >> 3, col = (e & 7) * 4, rc = row & 15, rtc = rc / p.group, t = t0 + (row >> 4) * tpt + rtc;
            if (rtc >= tpt || t >= p.queries) continue;
            f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < kWaves; ++w) sum += *reinterpret_cast<const f32x4 *>(merge + (w * RT * 16 + row) * kMergeStride + col);
            const int64_t at = ((int64_t)b * p.queries + t) * p.heads + h * p.group + (rc - rtc * p.group);
            const float2 st = joined[row];
            if (splits == 1) {
                const float inv = st.y == 0.f ? 0.f : 1.f / st.y;
                T *dst = out + at * D + strip * 32 + col;
#pragma unroll
                for (int i = 0; i < 4; ++i) dst[i] = (T)(sum[i] * inv);
                if (remainder)
#pragma unroll
                    for (int i = 0; i < 4; ++i) remainder[at * D + strip * 32 + col + i] = (T)(sum[i] * inv - (float)(T)(sum[i] * inv));
                if (strip == 0 && col == 0 && lse) lse[at] = st.y == 0.f ? __builtin_inff() : st.x + __builtin_amdgcn_logf(st.y);
            } else {
                *reinterpret_cast<f32x4 *>(part + (split * all_rows + at) * D + strip * 32 + col) = sum;
                if (strip == 0 && col == 0) part_stats[split * all_rows + at] = st;
            }
        }
    }
}

// Joins the sums of several workgroups per row: four columns a thread.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void block_attention_join_kernel(const float *part, const float2 *part_stats, T *out, T *remainder, float *lse, int64_t rows, int splits) {
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
#pragma unroll
    for (int i = 0; i < 4; ++i) out[row * D + col + i] = (T)(sum[i] * inv);
    if (remainder)
#pragma unroll
        for (int i = 0; i < 4; ++i) remainder[row * D + col + i] = (T)(sum[i] * inv - (float)(T)(sum[i] * inv));
    if (col == 0 && lse) lse[row] = total == 0.f ? __builtin_inff() : top + __builtin_amdgcn_logf(total);
}

// How many tiles of 16 rows a workgroup takes, and over how many workgroups a tile's list is dealt out.
struct Shape { int rt, n_tiles, splits; };
Shape shape_of(const Problem &p, int max_rt) {
    const int tpt = tile_tokens(p.group);
    const int64_t pairs = (int64_t)p.batch * p.kv_heads;
    Shape s{max_rt, 0, 1};
    auto tiles = [&](int rt) { return (p.queries + rt * tpt - 1) / (rt * tpt); };
    while (s.rt > 1 && pairs * tiles(s.rt) < 512) s.rt /= 2;
    s.n_tiles = tiles(s.rt);
    const int64_t groups = pairs * s.n_tiles;
    // units of a list at most; every wavefront keeps two of them
    const int64_t named = std::min<int64_t>((int64_t)p.topk * std::min(s.rt * tpt, p.queries), p.blocks);
    const int64_t units = named << (p.block_shift - 5);
    s.splits = (int)std::max<int64_t>(1, std::min<int64_t>((512 + groups - 1) / std::max<int64_t>(groups, 1), units / (2 * kWaves)));
    return s;
}

size_t round_up(size_t n) { return (n + 255) & ~(size_t)255; }

template <typename T, int D, int RT>
int launch_rt(const Problem &p, const Shape &s, T *out, T *rest, float *lse, float *part, float2 *part_stats, hipStream_t stream) {
    const size_t lds = stage_bytes<T, D, RT>() + buckets_bytes(p.n_buckets, p.low, p.high, p.group);
    const int64_t grid = (int64_t)p.batch * p.kv_heads * s.n_tiles * s.splits;
    if (grid >= (1ll << 31)) return fail(FG_ERR_SHAPE, "block attention: %lld workgroups do not fit a launch", (long long)grid);
    block_attention_kernel<T, D, RT><<<dim3((unsigned)grid), dim3(kThreads), lds, stream>>>(p, out, rest, lse, part, part_stats, s.n_tiles, s.splits);
    FG_HIP_TRY(hipGetLastError());
    return FG_OK;
}

template <typename T, int D> constexpr int max_row_tiles() { return sizeof(T) == 4 ? 2 : 4; }

template <typename T, int D>
int launch(const Problem &p, const fg_block_attention_args *a, void *workspace, size_t bytes, size_t *need, hipStream_t stream) {
    const Shape s = shape_of(p, max_row_tiles<T, D>());
    const size_t rows = (size_t)p.batch * p.queries * p.heads;
    const size_t sums = s.splits > 1 ? round_up(rows * s.splits * D * sizeof(float)) : 0, stats = s.splits > 1 ? round_up(rows * s.splits * sizeof(float2)) : 0;
    if (need) { *need = sums + stats; return FG_OK; }
    if (bytes < sums + stats || (sums && !workspace)) return fail(FG_ERR_ARG, "block attention: a workspace of %zu bytes, %zu needed (fg_block_attention_workspace)", bytes, sums + stats);
    float *part = static_cast<float *>(workspace);
    float2 *part_stats = reinterpret_cast<float2 *>(static_cast<unsigned char *>(workspace) + sums);
    T *out = static_cast<T *>(a->out), *rest = static_cast<T *>(a->rest);
    int rc;
    if constexpr (max_row_tiles<T, D>() == 4) {
        rc = s.rt == 4 ? launch_rt<T, D, 4>(p, s, out, rest, a->lse, part, part_stats, stream)
           : s.rt == 2 ? launch_rt<T, D, 2>(p, s, out, rest, a->lse, part, part_stats, stream)
                       : launch_rt<T, D, 1>(p, s, out, rest, a->lse, part, part_stats, stream);
    } else {
        rc = s.rt == 2 ? launch_rt<T, D, 2>(p, s, out, rest, a->lse, part, part_stats, stream) : launch_rt<T, D, 1>(p, s, out, rest, a->lse, part, part_stats, stream);
    }
    if (rc != FG_OK || s.splits == 1) return rc;
    const int64_t threads = (int64_t)rows * (D / 4);
    block_attention_join_kernel<T, D><<<dim3((unsigned)((threads + kThreads - 1) / kThreads)), dim3(kThreads), 0, stream>>>(part, part_stats, out, rest, a->lse, (int64_t)rows, s.splits);
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

int strides_of(const char *name, const void *ptr, const int64_t *stride, int size, Strides *s) {
    const int64_t per = 16 / size;
    if (reinterpret_cast<uintptr_t>(ptr) % 16 || stride[0] % per || stride[1] % per || stride[2] % per)
        return fail(FG_ERR_ARG, "block attention: %s and its strides have to be multiples of 16 bytes", name);
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
    if (a->keys > (1 << 30) || a->queries > (1 << 30) || (int64_t)a->topk * 64 > INT32_MAX / a->kv_heads)
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
        (rc = strides_of("v", a->v, a->v_strides, size, &p->vs))) return rc;
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
    return fg::block::launch_t(p, args, workspace, workspace_bytes, nullptr, static_cast<hipStream_t>(stream));
}
