// Gradients of attention over selected blocks of keys.  With p_ij = 2^(z_ij - lse_i) the forward pass's softmax:
//   dP_ij = <dO_i, V_j>,  dS_ij = p_ij (dP_ij - delta_i),  delta_i = <dO_i, O_i>
//   dQ_i = scale sum_j dS_ij K_j,  dK_j = scale sum_i dS_ij Q_i,  dV_j = sum_i p_ij dO_i,  dbias[n, h] = sum of dS_ij in bucket n
//
// Two sweeps form the scores again.  queries_kernel goes by query like the forward pass (its list of blocks, dQ and dbias).  keys_kernel goes by block:
// the lists are turned round -- for every block the tokens that selected it, in order -- and a workgroup takes a block, or a piece of a long
// list, with its keys in registers, and gathers the rows of its tokens' heads.  Nothing is added by atomics: sums over pieces,
// wavefronts and tiles are joined in a fixed order, so that a step gives the same bits every time.
#include <algorithm>
#include <type_traits>

#include "fg_block.h"

namespace fg {
namespace block {

namespace {

constexpr int kMergeStride = 36;       // floats between rows of the joining buffer (32 and 4 of padding)
constexpr int kPieceRows = 2048;       // rows (tokens times heads of the group) of one piece of a block's list

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

// Where each block's tokens, pieces and partial sums begin; totals[0]: all pieces.  One workgroup.
constexpr int kScan = 1024;
__global__ __launch_bounds__(kScan) void scan_kernel(const int32_t *count, int32_t *offset, int32_t *piece0, int32_t *slot0, int32_t *totals, int all, int piece) {
    __shared__ int sums[3][kScan / 64];
    int base[3] = {0, 0, 0};
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int m0 = 0; m0 < all; m0 += kScan) {
        const int m = m0 + tid, n = m < all ? count[m] : 0, k = (n + piece - 1) / piece;
        const int own[3] = {n, m < all ? max(k, 1) : 0, k > 1 ? k : 0};
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

// The tokens of every block in ascending order, and its pieces: one wavefront per block.
__global__ __launch_bounds__(kThreads) void fill_kernel(const unsigned long long *bits, const int32_t *count, const int32_t *offset, const int32_t *piece0,
                                                        const int32_t *slot0, int32_t *list, Piece *pieces, int all, int blocks, int chunks, int piece) {
    const int m = blockIdx.x * kWaves + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (m >= all) return;
    const int pair = m / blocks, n = count[m], k = max((n + piece - 1) / piece, 1), at0 = offset[m];
    for (int i = lane; i < k; i += 64) pieces[piece0[m] + i] = Piece{m, at0 + i * piece, min(piece, n - i * piece), k > 1 ? slot0[m] + i : -1};
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

template <typename T, int D, int RT> constexpr size_t queries_stage_bytes() {
    const size_t keys = (size_t)kWaves * kUnit * (D + kPad) * sizeof(T), merge = (size_t)kWaves * RT * 16 * kMergeStride * sizeof(float);
    return keys > merge ? keys : merge;
}

template <typename T, int D, int RT>
__global__ __launch_bounds__(kThreads) void queries_kernel(const Problem p, const T *dout, Strides ds, const T *out, const T *remainder, const float *lse, float *delta,
                                                           T *dq, float *bias_sums, int n_tiles) {
    constexpr int DC = D / 32, DT = D / 16, S = D + kPad;
    __shared__ List list;
    extern __shared__ __align__(16) unsigned char dynamic[];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, c = lane & 15;
    const int unit = xcd_contiguous_block(), pair = unit / n_tiles, tile = unit - pair * n_tiles;
    const int b = pair / p.kv_heads, h = pair - b * p.kv_heads;
    const int k_len = key_count(p, b), q_len = query_count(p, b), offset = k_len - q_len;
    const int tpt = tile_tokens(p.group), t0 = tile * RT * tpt, nt = RT * tpt;
    const int tc = c / p.group, mine = c - tc * p.group, head = h * p.group + mine;
    const bool used = tc < tpt;

    T *stage = reinterpret_cast<T *>(dynamic) + wave * kUnit * S;
    Buckets buckets;
    float *sums = nullptr;             // [bucket][lane] of this wavefront: a lane's rows all have one head
    if (p.n_buckets) {
        unsigned char *at = dynamic + queries_stage_bytes<T, D, RT>();
        buckets = load_buckets<T>(p, h, at);
        sums = reinterpret_cast<float *>(at + ((buckets_bytes(p.n_buckets, p.low, p.high, p.group) + 15) & ~(size_t)15)) + wave * p.n_buckets * 64;
    }

    V8<T> qf[RT][DC], df[RT][DC];
    int limit[RT];
    float row_lse[RT], row_delta[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int t = t0 + rt * tpt + tc;
        const bool there = used && t < q_len;
        limit[rt] = there ? (p.causal ? min(offset + t, k_len - 1) : k_len - 1) : used ? -1 : k_len - 1;
        const int64_t at = ((int64_t)b * p.queries + t) * p.heads + head;
        const T *qs = static_cast<const T *>(p.q) + b * p.qs.batch + (int64_t)t * p.qs.row + head * p.qs.head + 8 * g;
        const T *dos = dout + b * ds.batch + (int64_t)t * ds.row + head * ds.head + 8 * g, *os = out + at * D + 8 * g;
        float sum = 0.f;
#pragma unroll
        for (int dc = 0; dc < DC; ++dc) {
            qf[rt][dc] = there ? load8(qs + dc * 32) : zero8<T>();
            df[rt][dc] = there ? load8(dos + dc * 32) : zero8<T>();
            const V8<T> o = there ? load8(os + dc * 32) : zero8<T>();
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += (float)df[rt][dc][i] * (float)o[i];
            if (remainder) {
                const V8<T> r = there ? load8(remainder + at * D + 8 * g + dc * 32) : zero8<T>();
#pragma unroll
                for (int i = 0; i < 8; ++i) sum += (float)df[rt][dc][i] * (float)r[i];
            }
        }
        row_delta[rt] = rows_sum(sum);
        row_lse[rt] = there ? lse[at] : __builtin_inff();
        if (there && wave == 0 && g == 0) delta[at] = row_delta[rt];
    }
    const int last_key = p.causal ? min(k_len - 1, offset + min(t0 + nt, q_len) - 1) : k_len - 1;
    const T *kbase = static_cast<const T *>(p.k) + b * p.ks.batch + h * p.ks.head + 8 * g;
    const T *vbase = static_cast<const T *>(p.v) + b * p.vs.batch + h * p.vs.head + 8 * g;
    const int sub_shift = p.block_shift - 5;

    f32x4 acc[RT][DT];
    auto sweep = [&](auto careful) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) acc[rt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int n = 0; n < p.n_buckets; ++n) sums[n * 64 + lane] = 0.f;
        for (int first = 0; first < p.blocks; first += kWindow) {
            const int units = build_list(list, p, b, h, t0, nt, q_len, k_len, first, min(kWindow, p.blocks - first)) << sub_shift;
            auto first_key = [&](int u) {
                return __builtin_amdgcn_readfirstlane(((first + list.id[u >> sub_shift]) << p.block_shift) + ((u & ((1 << sub_shift) - 1)) << 5));
            };
            auto find = [&](int u) {
                while (u < units && first_key(u) > last_key) u += kWaves;
                return u;
            };
            V8<T> kf[2][DC], vf[2][DC];
            int key0 = 0;
            unsigned long long bits = 0;
            auto fetch = [&](int u) {
                key0 = first_key(u);
                bits = uniform64(list.bits[u >> sub_shift]);
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
                const int now = key0;
                const unsigned long long who = bits;
                wave_lds_sync();
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int dc = 0; dc < DC; ++dc) *reinterpret_cast<V8<T> *>(stage + (kt * 16 + c) * S + dc * 32 + 8 * g) = kf[kt][dc];
                wave_lds_sync();
                f32x4 s[RT][2], dp[RT][2];
                unsigned active = 0;
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    if (!((who >> (rt * tpt)) & ((1ull << tpt) - 1))) continue;
                    active |= 1u << rt;
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt) {
                        s[rt][kt] = dp[rt][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int dc = 0; dc < DC; ++dc) {
                            s[rt][kt] = mma(kf[kt][dc], qf[rt][dc], s[rt][kt]);
                            dp[rt][kt] = mma(vf[kt][dc], df[rt][dc], dp[rt][kt]);
                        }
                    }
                }
                u = find(u + kWaves);
                if (u < units) fetch(u);

                V8<T> pf[RT];
                unsigned seen[RT];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    if (!(active & (1u << rt))) continue;
                    const int last = !used || (who >> (rt * tpt + tc)) & 1 ? limit[rt] : -1;
                    const int pos = offset + t0 + rt * tpt;
                    const int near = p.n_buckets ? buckets.at(pos - now - (kUnit - 1)) : 0, far = p.n_buckets ? buckets.at(pos + tpt - 1 - now) : 0;
                    unsigned mask = 0;
                    float total = 0.f;
                    const float common = p.n_buckets && near == far ? buckets.value(near, mine) : 0.f;
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int key = now + 16 * kt + 4 * g + i;
                            const bool ok = key <= last;
                            float z = s[rt][kt][i] * p.scale2 + common;
                            int bucket = 0;
                            if (near != far) {
                                bucket = buckets.at(pos + tc - key);
                                z += buckets.value(bucket, mine);
                            }
                            const float x = __builtin_amdgcn_exp2f(z - row_lse[rt]) * (dp[rt][kt][i] - row_delta[rt]);
                            s[rt][kt][i] = ok ? x : 0.f;
                            mask |= (unsigned)ok << (4 * kt + i);
                            if (near != far) sums[bucket * 64 + lane] += s[rt][kt][i];
                            else total += s[rt][kt][i];
                        }
                    if (p.n_buckets && near == far) sums[near * 64 + lane] += total;
                    seen[rt] = mask;
                    // rounded to the operands' type for the product with K, half a step each
                    pf[rt] = pack<T>(s[rt][0], s[rt][1]);
                }
                if (!careful && active == (1u << RT) - 1) {
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) {
                        const V8<T> x = transposed<T, D>(stage, dt * 16, lane);
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt) acc[rt][dt] = mma(x, pf[rt], acc[rt][dt]);
                    }
                } else {
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        if (!(active & (1u << rt))) continue;
#pragma unroll
                        for (int dt = 0; dt < DT; ++dt) {
                            const V8<T> x = transposed<T, D>(stage, dt * 16, lane);
                            if constexpr (decltype(careful)::value) acc[rt][dt] = mma_masked<T>(x, pf[rt], seen[rt], acc[rt][dt]);
                            else acc[rt][dt] = mma(x, pf[rt], acc[rt][dt]);
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
        for (int dt = 0; dt < DT; ++dt) odd |= not_finite(acc[rt][dt]);
    if (__syncthreads_or(odd)) sweep(std::true_type{});

    float *merge = reinterpret_cast<float *>(dynamic);
#pragma unroll
    for (int strip = 0; strip < DC; ++strip) {
        __syncthreads();               // the keys' staging, or the strip before, has been read
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                *reinterpret_cast<f32x4 *>(merge + ((wave * RT + rt) * 16 + c) * kMergeStride + 16 * j + 4 * g) = acc[rt][2 * strip + j];
        __syncthreads();
        for (int e = tid; e < RT * 16 * 8; e += kThreads) {
            const int row = e >> 3, col = (e & 7) * 4, rc = row & 15, rtc = rc / p.group, t = t0 + (row >> 4) * tpt + rtc;
            if (rtc >= tpt || t >= p.queries) continue;
            f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < kWaves; ++w) sum += *reinterpret_cast<const f32x4 *>(merge + (w * RT * 16 + row) * kMergeStride + col);
            T *dst = dq + (((int64_t)b * p.queries + t) * p.heads + h * p.group + (rc - rtc * p.group)) * D + strip * 32 + col;
#pragma unroll
            for (int i = 0; i < 4; ++i) dst[i] = (T)(sum[i] * p.scale);
        }
    }
    if (p.n_buckets) {                 // the tile's share of the bias's gradient, [sequence and tile][head][bucket]
        sums -= wave * p.n_buckets * 64;
        for (int e = tid; e < p.n_buckets * p.group; e += kThreads) {
            const int x = e / p.n_buckets, n = e - x * p.n_buckets;
            float total = 0.f;
            for (int w = 0; w < kWaves; ++w)
                for (int t = 0; t < tpt; ++t)
                    for (int q = 0; q < 4; ++q) total += sums[(w * p.n_buckets + n) * 64 + q * 16 + t * p.group + x];
            bias_sums[(((int64_t)b * n_tiles + tile) * p.heads + h * p.group + x) * p.n_buckets + n] = total;
        }
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

// A wavefront has 32 keys; where a block has fewer than 4 x 32, several wavefronts share them and take the list's rows in turn.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void keys_kernel(const Problem p, const T *dout, Strides ds, const float *lse, const float *delta, const Piece *pieces,
                                                        const int32_t *totals, const int32_t *list, float *partial, T *dk, T *dv) {
    constexpr int DC = D / 32, DT = D / 16, S = D + kPad;
    struct Row { float lse, delta; int pos, head; };
    __shared__ Row rows[kWaves][kUnit];
    extern __shared__ __align__(16) unsigned char dynamic[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, c = lane & 15;
    const int block = 1 << p.block_shift, kw_n = min(kWaves, block / kUnit), rw_n = kWaves / kw_n, parts = block / (kw_n * kUnit);
    const int kw = wave % kw_n, rw = wave / kw_n, work = blockIdx.x / parts, part = blockIdx.x - work * parts;
    if (work >= totals[0]) return;
    const Piece piece = pieces[work];
    const int pair = piece.block / p.blocks, blk = piece.block - pair * p.blocks, b = pair / p.kv_heads, h = pair - b * p.kv_heads;
    const int k_len = key_count(p, b), q_len = query_count(p, b), offset = k_len - q_len;
    const int in_block = (part * kw_n + kw) * kUnit, key0 = (blk << p.block_shift) + in_block, n_rows = piece.len * p.group;

    T *stage_q = reinterpret_cast<T *>(dynamic) + wave * 2 * kUnit * S, *stage_d = stage_q + kUnit * S;
    Buckets buckets;
    if (p.n_buckets) {
        buckets = load_buckets<T>(p, h, dynamic + keys_stage_bytes<T, D>());
        __syncthreads();
    }

    V8<T> kf[2][DC], vf[2][DC];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
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
    const T *qbase = static_cast<const T *>(p.q) + b * p.qs.batch + (int64_t)h * p.group * p.qs.head + 8 * g;
    const T *dbase = dout + b * ds.batch + (int64_t)h * p.group * ds.head + 8 * g;
    Row *own = rows[wave];

    f32x4 ak[2][DT], av[2][DT];
    auto sweep = [&](auto careful) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) ak[kt][dt] = av[kt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
        V8<T> qf[2][DC], df[2][DC];
        Row next;                      // lane 16 rt + c: row 16 rt + c of the step
        auto fetch = [&](int r0) {
            const int r = r0 + (lane & 31);
            const bool there = r < n_rows;
            int token = 0, x = 0;
            next = Row{__builtin_inff(), 0.f, -1, 0};
            if (there) {
                const int at = r / p.group;
                x = r - at * p.group;
                token = list[piece.start + at];
                const int64_t row = ((int64_t)b * p.queries + token) * p.heads + h * p.group + x;
                next = Row{lse[row], delta[row], offset + token, x};
            }
#pragma unroll
            for (int rt = 0; rt < 2; ++rt) {
                const int t = __shfl(token, rt * 16 + c), y = __shfl(x, rt * 16 + c);
                const bool ok = r0 + rt * 16 + c < n_rows;
                const T *q = qbase + (int64_t)t * p.qs.row + y * p.qs.head, *d = dbase + (int64_t)t * ds.row + y * ds.head;
#pragma unroll
                for (int dc = 0; dc < DC; ++dc) {
                    qf[rt][dc] = ok ? load8(q + dc * 32) : zero8<T>();
                    df[rt][dc] = ok ? load8(d + dc * 32) : zero8<T>();
                }
            }
        };
        int r0 = rw * kUnit;
        if (r0 < n_rows) fetch(r0);
        while (r0 < n_rows) {
            wave_lds_sync();
#pragma unroll
            for (int rt = 0; rt < 2; ++rt)
#pragma unroll
                for (int dc = 0; dc < DC; ++dc) {
                    *reinterpret_cast<V8<T> *>(stage_q + (rt * 16 + c) * S + dc * 32 + 8 * g) = qf[rt][dc];
                    *reinterpret_cast<V8<T> *>(stage_d + (rt * 16 + c) * S + dc * 32 + 8 * g) = df[rt][dc];
                }
            if (lane < kUnit) own[lane] = next;
            wave_lds_sync();
            f32x4 s[2][2], dp[2][2];   // [rows][keys]
#pragma unroll
            for (int rt = 0; rt < 2; ++rt)
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) {
                    s[rt][kt] = dp[rt][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int dc = 0; dc < DC; ++dc) {
                        s[rt][kt] = mma(qf[rt][dc], kf[kt][dc], s[rt][kt]);
                        dp[rt][kt] = mma(df[rt][dc], vf[kt][dc], dp[rt][kt]);
                    }
                }
            r0 += rw_n * kUnit;
            if (r0 < n_rows) fetch(r0);

            unsigned seen[2] = {0, 0};
#pragma unroll
            for (int rt = 0; rt < 2; ++rt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const Row row = own[rt * 16 + 4 * g + i];
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt) {
                        const int key = key0 + kt * 16 + c;
                        const bool ok = key <= (p.causal ? row.pos : k_len - 1);     // a row behind the last has no weight: lse is inf
                        float z = s[rt][kt][i] * p.scale2;
                        if (p.n_buckets) z += buckets.value(buckets.at(row.pos - key), row.head);
                        const float x = ok ? __builtin_amdgcn_exp2f(z - row.lse) : 0.f;
                        s[rt][kt][i] = x;
                        dp[rt][kt][i] = ok ? x * (dp[rt][kt][i] - row.delta) : 0.f;
                        seen[kt] |= (unsigned)ok << (4 * rt + i);
                    }
                }
            V8<T> pf[2], sf[2];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                pf[kt] = pack<T>(s[0][kt], s[1][kt]);
                sf[kt] = pack<T>(dp[0][kt], dp[1][kt]);
            }
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const V8<T> d = transposed<T, D>(stage_d, dt * 16, lane), q = transposed<T, D>(stage_q, dt * 16, lane);
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) {
                    if constexpr (decltype(careful)::value) {
                        av[kt][dt] = mma_masked<T>(d, pf[kt], seen[kt], av[kt][dt]);
                        ak[kt][dt] = mma_masked<T>(q, sf[kt], seen[kt], ak[kt][dt]);
                    } else {
                        av[kt][dt] = mma(d, pf[kt], av[kt][dt]);
                        ak[kt][dt] = mma(q, sf[kt], ak[kt][dt]);
                    }
                }
            }
        }
    };
    sweep(std::false_type{});
    bool odd = false;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) odd |= not_finite(ak[kt][dt]) || not_finite(av[kt][dt]);
    if (__any(odd)) sweep(std::true_type{});

    // wavefronts that share keys: the upper half hands its sums to the lower one, until one has them all
    f32x4 *merge = reinterpret_cast<f32x4 *>(dynamic);
    for (int half = rw_n >> 1; half; half >>= 1) {
        __syncthreads();
        if (rw >= half && rw < 2 * half) {
            f32x4 *to = merge + ((rw - half) * kw_n + kw) * (4 * DT * 64) + lane;
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) { to[(kt * DT + dt) * 128] = ak[kt][dt]; to[(kt * DT + dt) * 128 + 64] = av[kt][dt]; }
        }
        __syncthreads();
        if (rw < half) {
            const f32x4 *from = merge + (rw * kw_n + kw) * (4 * DT * 64) + lane;
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) { ak[kt][dt] += from[(kt * DT + dt) * 128]; av[kt][dt] += from[(kt * DT + dt) * 128 + 64]; }
        }
    }
    if (rw) return;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
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

// Blocks whose lists were cut: the pieces' sums, in order.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void pieces_kernel(const Problem p, const int32_t *count, const int32_t *slot0, const float *partial, T *dk, T *dv, int piece) {
    const int m = blockIdx.x, k = (count[m] + piece - 1) / piece;
    if (k <= 1) return;
    const int pair = m / p.blocks, blk = m - pair * p.blocks, b = pair / p.kv_heads, h = pair - b * p.kv_heads, block = 1 << p.block_shift;
    const float *src = partial + (int64_t)slot0[m] * 2 * block * D;
    for (int e = threadIdx.x; e < 2 * block * (D / 4); e += kThreads) {
        const int row = e / (D / 4), col = (e - row * (D / 4)) * 4, key = (blk << p.block_shift) + (row & (block - 1));
        if (key >= p.keys) continue;
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
        for (int i = 0; i < k; ++i) sum += *reinterpret_cast<const f32x4 *>(src + ((int64_t)i * 2 * block + row) * D + col);
        T *dst = (row < block ? dk : dv) + (((int64_t)b * p.keys + key) * p.kv_heads + h) * D + col;
        const float scale = row < block ? p.scale : 1.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) dst[i] = (T)(sum[i] * scale);
    }
}

// ---- host -------------------------------------------------------------------------------------------------

struct Layout {
    int rt, n_tiles, chunks, piece;
    int64_t all, pieces, slots, entries;       // blocks of all sequences and key heads; bounds on the others
    size_t delta, bits, count, offset, piece0, slot0, totals, list, table, partial, bias, bytes;
};

int layout_of(const Problem &p, int head_len, int max_rt, Layout *l) {
    const int tpt = tile_tokens(p.group);
    const int64_t pairs = (int64_t)p.batch * p.kv_heads;
    auto tiles = [&](int rt) { return (p.queries + rt * tpt - 1) / (rt * tpt); };
    l->rt = max_rt;
    while (l->rt > 1 && pairs * tiles(l->rt) < 512) l->rt /= 2;
    l->n_tiles = tiles(l->rt);
    l->chunks = std::max(1, (p.queries + 63) / 64);
    l->piece = std::max(1, kPieceRows / p.group);
    l->all = pairs * p.blocks;
    l->entries = pairs * p.queries * std::min(p.topk, p.blocks);
    l->pieces = l->all + l->entries / l->piece;
    l->slots = 2 * (l->entries / l->piece);
    const int64_t limit = INT32_MAX;
    if (l->entries > limit || l->pieces * 2 > limit || pairs * std::max(l->n_tiles, l->chunks) > limit)
        return fail(FG_ERR_SHAPE, "block attention gradients: %lld selections do not fit the 32-bit lists", (long long)l->entries);
    size_t at = 0;
    auto place = [&](size_t n) { const size_t here = at; at += (n + 255) & ~(size_t)255; return here; };
    l->delta = place((size_t)p.batch * p.queries * p.heads * sizeof(float));
    l->bits = place((size_t)l->all * l->chunks * 8);
    l->count = place((size_t)l->all * 4);
    l->offset = place((size_t)l->all * 4);
    l->piece0 = place((size_t)l->all * 4);
    l->slot0 = place((size_t)l->all * 4);
    l->totals = place(4);
    l->list = place((size_t)l->entries * 4);
    l->table = place((size_t)l->pieces * sizeof(Piece));
    l->partial = place((size_t)l->slots * 2 * ((size_t)1 << p.block_shift) * head_len * sizeof(float));
    l->bias = place((size_t)p.batch * l->n_tiles * p.heads * p.n_buckets * sizeof(float));
    l->bytes = at;
    return FG_OK;
}

template <typename T, int D, int RT>
int launch_queries(const Problem &p, const Layout &l, const fg_block_attention_args *a, const fg_block_attention_grads *grads, Strides ds, unsigned char *w, hipStream_t stream) {
    size_t lds = queries_stage_bytes<T, D, RT>();
    if (p.n_buckets) lds += ((buckets_bytes(p.n_buckets, p.low, p.high, p.group) + 15) & ~(size_t)15) + (size_t)kWaves * p.n_buckets * 64 * sizeof(float);
    queries_kernel<T, D, RT><<<dim3((unsigned)(p.batch * p.kv_heads * l.n_tiles)), dim3(kThreads), lds, stream>>>(
        p, static_cast<const T *>(grads->dout), ds, static_cast<const T *>(a->out), static_cast<const T *>(a->rest), a->lse, reinterpret_cast<float *>(w + l.delta),
        static_cast<T *>(grads->dq), reinterpret_cast<float *>(w + l.bias), l.n_tiles);
    FG_HIP_TRY(hipGetLastError());
    return FG_OK;
}

template <typename T, int D>
int launch(const Problem &p, const fg_block_attention_args *a, const fg_block_attention_grads *grads, void *workspace, size_t bytes, size_t *need, hipStream_t stream) {
    Layout l;
    if (int rc = layout_of(p, D, sizeof(T) == 4 || D == 128 ? 2 : 4, &l)) return rc;
    if (need) { *need = l.bytes; return FG_OK; }
    if (bytes < l.bytes || (l.bytes && !workspace)) return fail(FG_ERR_ARG, "block attention gradients: a workspace of %zu bytes, %zu needed (fg_block_attention_backward_workspace)", bytes, l.bytes);
    Strides ds;
    if (int rc = strides_of("dout", grads->dout, grads->dout_strides, sizeof(T), &ds)) return rc;
    unsigned char *w = static_cast<unsigned char *>(workspace);
    int rc = FG_OK;
    if (p.queries == 0) {
    } else if constexpr (sizeof(T) == 4 || D == 128)
        rc = l.rt == 2 ? launch_queries<T, D, 2>(p, l, a, grads, ds, w, stream) : launch_queries<T, D, 1>(p, l, a, grads, ds, w, stream);
    else
        rc = l.rt == 4 ? launch_queries<T, D, 4>(p, l, a, grads, ds, w, stream)
           : l.rt == 2 ? launch_queries<T, D, 2>(p, l, a, grads, ds, w, stream) : launch_queries<T, D, 1>(p, l, a, grads, ds, w, stream);
    if (rc != FG_OK) return rc;
    if (p.n_buckets && grads->dbias) {
        bias_kernel<T><<<dim3(p.heads), dim3(1024), 0, stream>>>(reinterpret_cast<const float *>(w + l.bias), static_cast<T *>(grads->dbias), p.batch * l.n_tiles, p.heads, p.n_buckets);
        FG_HIP_TRY(hipGetLastError());
    }
    if (!grads->dk || l.all == 0) return FG_OK;
    auto bits = reinterpret_cast<unsigned long long *>(w + l.bits);
    auto ints = [&](size_t at) { return reinterpret_cast<int32_t *>(w + at); };
    auto pieces = reinterpret_cast<Piece *>(w + l.table);
    const int all = (int)l.all, per_wave = (all + kWaves - 1) / kWaves, block = 1 << p.block_shift, parts = std::max(1, block / (kWaves * kUnit));
    mark_kernel<<<dim3((unsigned)(p.batch * p.kv_heads * l.chunks)), dim3(kThreads), 0, stream>>>(p, bits, l.chunks);
    count_kernel<<<dim3(per_wave), dim3(kThreads), 0, stream>>>(bits, ints(l.count), all, p.blocks, l.chunks);
    scan_kernel<<<dim3(1), dim3(kScan), 0, stream>>>(ints(l.count), ints(l.offset), ints(l.piece0), ints(l.slot0), ints(l.totals), all, l.piece);
    fill_kernel<<<dim3(per_wave), dim3(kThreads), 0, stream>>>(bits, ints(l.count), ints(l.offset), ints(l.piece0), ints(l.slot0), ints(l.list), pieces, all, p.blocks, l.chunks, l.piece);
    const size_t lds = keys_stage_bytes<T, D>() + buckets_bytes(p.n_buckets, p.low, p.high, p.group);
    keys_kernel<T, D><<<dim3((unsigned)(l.pieces * parts)), dim3(kThreads), lds, stream>>>(
        p, static_cast<const T *>(grads->dout), ds, a->lse, reinterpret_cast<const float *>(w + l.delta), pieces, ints(l.totals), ints(l.list),
        reinterpret_cast<float *>(w + l.partial), static_cast<T *>(grads->dk), static_cast<T *>(grads->dv));
    if (l.slots)
        pieces_kernel<T, D><<<dim3(all), dim3(kThreads), 0, stream>>>(p, ints(l.count), ints(l.slot0), reinterpret_cast<const float *>(w + l.partial),
                                                                      static_cast<T *>(grads->dk), static_cast<T *>(grads->dv), l.piece);
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
    if (p.batch == 0) return FG_OK;
    if ((p.queries && (!p.q || !p.list || !args->out || !args->lse || !grads->dout || !grads->dq)) || (p.keys && (!p.k || !p.v)) ||
        !grads->dk != !grads->dv || (p.n_buckets && !p.bias))
        return fg::fail(FG_ERR_ARG, "block attention gradients: null pointer");
    return fg::block::launch_t(p, args, grads, workspace, workspace_bytes, nullptr, static_cast<hipStream_t>(stream));
}
