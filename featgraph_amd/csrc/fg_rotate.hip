// RMS norm of every head of queries and keys, and their rotation by position, in one pass; and its gradients.
//   xh = x / sqrt(mean(x^2) + eps),  y = w xh (or x where there are no weights),  each pair (a, b) of the first rotary_len elements of y turned by
//   t = 2 pi position[axis(pair)] turns[pair]:  (a cos t - b sin t, a sin t + b cos t);  pairs are (i, i + rotary_len / 2) or neighbours.
//   Gradients: g = w (dout turned by -t),  dx = (g - xh mean(g xh)) / sqrt(mean(x^2) + eps),  dw = sum over all rows of xh (dout turned by -t).
//
// Angles are products in 64 bits, less their whole turns before they are rounded: a position of 10^6 has as good a sine as position 1.  What that rounding takes, l, follows
// in cos - l sin and sin + l cos.  A wavefront makes a token's sines once, a pair a lane, and takes them from LDS for all its heads.
// A lane holds one 16-byte piece of each half of a head's pairs, so that partners need no exchange; elements that are not turned
// (rotary_len < head_len) are dealt to the halves the same way.
// Sums in 32 bits; dw's sums over rows in 32 bits per wavefront and 64 after that, for 32-bit results in 32 bits for 16 rows of a lane and 64 after that.
//
// What bounds them.  16,384 tokens of 32 / 8 heads of 128 in bfloat16: 67 us, 5.0 TB/s, the rate of a large copy; gradients of 2 x 4,096 tokens of 16 / 4
// heads 29.6 us, 4.3 TB/s (three wavefronts a SIMD: 32 sums, two heads' elements and the next ones' take 168 registers), their weights' sums 4. One token
// each of 32 sequences 3.4 us: the chain lengths, angles, LDS, store.
#include <algorithm>

#include "fg_block.h"

namespace fg {
namespace rotate {

namespace {

using block::Strides;

constexpr int kWaves = 4, kThreads = 64 * kWaves, kPairs = 64;

struct Problem {
    int batch, tokens, heads, kv_heads, rotary_len, interleaved, axes, parts;
    float eps;
    const void *q, *k, *q_weight, *k_weight;
    Strides qs, ks;
    const int32_t *positions, *lengths, *q_lengths;
    double turns[kPairs];              // of a pair and a position
    uint8_t axis[kPairs];
};

template <typename T> struct Piece;                   // 16 bytes
template <> struct Piece<float> { static constexpr int N = 4; typedef float V __attribute__((ext_vector_type(4))); };
template <> struct Piece<_Float16> { static constexpr int N = 8; typedef _Float16 V __attribute__((ext_vector_type(8))); };
template <> struct Piece<__bf16> { static constexpr int N = 8; typedef __bf16 V __attribute__((ext_vector_type(8))); };

// What a lane holds of a head: E elements from `a` on and E from `b` on, and where their sines stand.
template <typename T, int D> struct Lane {
    static constexpr int E = Piece<T>::N, kLanes = D / 2 / E, kHeads = 64 / kLanes;      // lanes of a head; heads of a wavefront at a time
    int slot, a, b, first[2];
    bool turned;
    __device__ __forceinline__ Lane(const Problem &p, int lane) {
        const int half = p.rotary_len / 2, at = lane % kLanes * E;
        slot = lane / kLanes;
        turned = at < half;
        a = turned ? at : p.rotary_len + at - half;
        b = turned ? half + at : p.rotary_len + (D - p.rotary_len) / 2 + at - half;
        first[0] = p.interleaved ? a / 2 : at;
        first[1] = p.interleaved ? b / 2 : at + E / 2;
    }
};

// A token's cosines and sines, for all lanes of a wavefront.
__device__ __forceinline__ void make_angles(const Problem &p, int b, int i, int q_len, int lane, float2 *table) {
    wave_lds_sync();                   // of the token before
    if (lane < p.rotary_len / 2) {
        int64_t position;
        if (p.positions) position = p.positions[((int64_t)b * p.tokens + i) * p.axes + p.axis[lane]];
        else position = (int64_t)(p.lengths ? p.lengths[b] : q_len) - q_len + i;
        double t = (double)position * p.turns[lane];
        t = 2.0 * (t - rint(t));
        const float near = (float)t, rest = (float)((t - (double)near) * 3.14159265358979323846);      // what rounding takes from an angle
        float2 cs;
        sincospif(near, &cs.y, &cs.x);
        table[lane] = make_float2(cs.x - rest * cs.y, cs.y + rest * cs.x);
    }
    wave_lds_sync();
}

// (a, b) of one lane turned; sign -1: back.
template <typename T, int D>
__device__ __forceinline__ void turn(const Problem &p, const Lane<T, D> &me, const float2 *cs, float sign, float (&a)[Piece<T>::N], float (&b)[Piece<T>::N]) {
    constexpr int E = Piece<T>::N;
    if (!me.turned) return;
    if (p.interleaved) {
#pragma unroll
        for (int i = 0; i < E / 2; ++i) {
            const float c0 = cs[i].x, s0 = sign * cs[i].y, c1 = cs[E / 2 + i].x, s1 = sign * cs[E / 2 + i].y;
            const float x = a[2 * i], y = b[2 * i];
            a[2 * i] = x * c0 - a[2 * i + 1] * s0;
            a[2 * i + 1] = x * s0 + a[2 * i + 1] * c0;
            b[2 * i] = y * c1 - b[2 * i + 1] * s1;
            b[2 * i + 1] = y * s1 + b[2 * i + 1] * c1;
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float x = a[i], s = sign * cs[i].y;
            a[i] = x * cs[i].x - b[i] * s;
            b[i] = x * s + b[i] * cs[i].x;
        }
    }
}

template <int L> __device__ __forceinline__ float lanes_sum(float v) {
    if constexpr (L == 2) return v + dpp_move<0xB1>(v);
    else return group_sum<L>(v);
}

// 1 / sqrt(mean(x^2) + eps) over a head's lanes.  Where squares leave the range of 32 bits the elements are scaled by a power of two, `by`, first, in
// place: the result is that of the scaled ones, and `by` times it that of the elements.
template <typename T, int D>
__device__ __forceinline__ float inverse_rms(float (&a)[Piece<T>::N], float (&b)[Piece<T>::N], float eps, float *by) {
    constexpr int E = Piece<T>::N;
    auto sum = [&]() {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) s += a[i] * a[i] + b[i] * b[i];
        return lanes_sum<Lane<T, D>::kLanes>(s);
    };
    *by = 1.f;
    float s = sum();
    // small squares are lost beside any eps that is not small itself.  2^90 brings the smallest number there is to 2^-59 and leaves those that are small here, and eps, below 2^60
    const bool large = !(s < __builtin_inff()), small = s < 0x1p-100f && eps < 0x1p-60f;
    if (__any(large || small)) {
        *by = large ? 0x1p-70f : small ? 0x1p90f : 1.f;
#pragma unroll
        for (int i = 0; i < E; ++i) { a[i] *= *by; b[i] *= *by; }
        const float t = sum();
        s = large || small ? t : s;    // the others keep their sum to the bit, whoever stands beside them
    }
    return 1.f / sqrtf(s * (1.f / D) + eps * *by * *by);
}

// What a lane holds of a head, as it is stored.
template <typename T> struct Pair {
    typename Piece<T>::V a = {}, b = {};
    __device__ __forceinline__ void load(const T *pa, const T *pb) {
        a = *reinterpret_cast<const typename Piece<T>::V *>(pa);
        b = *reinterpret_cast<const typename Piece<T>::V *>(pb);
    }
    __device__ __forceinline__ void widen(float (&x)[Piece<T>::N], float (&y)[Piece<T>::N]) const {
#pragma unroll
        for (int i = 0; i < Piece<T>::N; ++i) { x[i] = (float)a[i]; y[i] = (float)b[i]; }
    }
};
template <typename T> __device__ __forceinline__ void put(T *p, const float (&f)[Piece<T>::N]) {
    typename Piece<T>::V v;
#pragma unroll
    for (int i = 0; i < Piece<T>::N; ++i) v[i] = (T)f[i];
    *reinterpret_cast<typename Piece<T>::V *>(p) = v;
}

// The sines of a lane's elements.
template <typename T, int D> __device__ __forceinline__ void own_angles(const Lane<T, D> &me, const float2 *table, float2 (&cs)[Piece<T>::N]) {
    constexpr int E = Piece<T>::N;
#pragma unroll
    for (int i = 0; i < E; ++i) cs[i] = me.turned ? table[me.first[i / (E / 2)] + i % (E / 2)] : make_float2(1.f, 0.f);
}

// A wavefront's share: one token, and every `parts`-th group of its heads.  A head's elements are under way while the one before is worked on, the first
// ones while angles are made.
template <typename T, int D, bool NORM>
__global__ __launch_bounds__(kThreads) void rotate_kernel(const Problem p, T *q_out, T *k_out) {
    constexpr int E = Piece<T>::N;
    __shared__ float2 table[kWaves][kPairs];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t unit = (int64_t)blockIdx.x * kWaves + wave, token = unit / p.parts;
    if (token >= (int64_t)p.batch * p.tokens) return;
    const int part = (int)(unit - token * p.parts), b = (int)(token / p.tokens), i = (int)(token - (int64_t)b * p.tokens);
    const int q_len = p.q_lengths ? min(max(p.q_lengths[b], 0), p.tokens) : p.tokens;
    const bool there = i < q_len;
    const Lane<T, D> me(p, lane);
    // heads of queries, then of keys: group g of kHeads heads is one wavefront's at a time
    const int q_groups = (p.heads + me.kHeads - 1) / me.kHeads, groups = q_groups + (p.kv_heads + me.kHeads - 1) / me.kHeads;
    const T *q = static_cast<const T *>(p.q) + b * p.qs.batch + (int64_t)i * p.qs.row, *k = static_cast<const T *>(p.k) + b * p.ks.batch + (int64_t)i * p.ks.row;
    Pair<T> next, weight;
    int h;                             // of the group that is under way
    auto fetch = [&](int group) {
        const bool keys = group >= q_groups;
        h = (keys ? group - q_groups : group) * me.kHeads + me.slot;
        if (!there || h >= (keys ? p.kv_heads : p.heads)) return;
        const T *src = keys ? k + h * p.ks.head : q + h * p.qs.head;
        next.load(src + me.a, src + me.b);
    };
    auto weigh = [&](int group) {
        const T *w = static_cast<const T *>(group >= q_groups ? p.k_weight : p.q_weight);
        if (NORM) weight.load(w + me.a, w + me.b);
    };
    fetch(part);
    weigh(part);
    float2 cs[E];
    if (there) {
        make_angles(p, b, i, q_len, lane, table[wave]);
        own_angles<T, D>(me, table[wave], cs);
    }
    for (int group = part; group < groups; group += p.parts) {
        const bool keys = group >= q_groups;
        const int now = h, heads = keys ? p.kv_heads : p.heads;
        float x[E], y[E];
        next.widen(x, y);
        if (group + p.parts < groups) fetch(group + p.parts);
        if (there) {
            if (NORM) {
                float wa[E], wb[E];
                weight.widen(wa, wb);
                float by;
                const float r = inverse_rms<T, D>(x, y, p.eps, &by);
#pragma unroll
                for (int e = 0; e < E; ++e) { x[e] = x[e] * r * wa[e]; y[e] = y[e] * r * wb[e]; }
            }
            turn<T, D>(p, me, cs, 1.f, x, y);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = y[e] = 0.f;
        }
        if (now < heads) {
            T *dst = (keys ? k_out : q_out) + (token * heads + now) * D;
            put(dst + me.a, x);
            put(dst + me.b, y);
        }
        if (!keys && group + p.parts >= q_groups) weigh(group + p.parts);
    }
}

struct Grads { const void *dq_out, *dk_out; Strides dqs, dks; void *dq, *dk; float *sums; };

// Workgroups of a CU (wavefronts of a SIMD) that registers are left for.
template <typename T, bool NORM> constexpr int kResident = NORM && sizeof(T) == 2 ? 3 : 4;
// dw's sums: a wavefront's in 64 bits for results of 32, to which a lane's go after every token that ends sixteen rows or more, through LDS.  Gradients of 3 x 1,237 tokens of 6 / 2 heads of 64 12.6 us with the
// weights' sums (with shuffles of 32-bit sums, one a wavefront, 13.7; of 64-bit ones 14.9), 64 x 8,192 of 4 / 4 heads of 32 567 (562); lanes with 64-bit sums take
// three wavefronts a SIMD and 14.6 and 671.  16-bit results are rounded by more than all of it.
template <typename T> using Sum = typename std::conditional<sizeof(T) == 4, double, float>::type;
template <typename T> constexpr int kRows = sizeof(T) == 4 ? 16 : 0;

// The same with the gradients; wavefronts take one token after the other and keep their share of dw: sums[workgroup][q, k][D].
template <typename T, int D, bool NORM>
__global__ __launch_bounds__(kThreads, (kResident<T, NORM>)) void rotate_backward_kernel(const Problem p, const Grads grads) {
    constexpr int E = Piece<T>::N;
    __shared__ float2 table[kWaves][kPairs];
    __shared__ Sum<T> shares[kWaves][2][D];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Lane<T, D> me(p, lane);
    float sum[2][2][E] = {};
    // 32-bit results: the lanes' sums into the wavefront's, by way of LDS
    __shared__ __align__(16) float parts[kRows<T> ? kWaves : 1][Lane<T, D>::kHeads][2][D];
    auto collect = [&]() {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                parts[wave][me.slot][k][me.a + e] = sum[k][0][e];
                parts[wave][me.slot][k][me.b + e] = sum[k][1][e];
                sum[k][0][e] = sum[k][1][e] = 0.f;
            }
        }
        wave_lds_sync();
#pragma unroll
        for (int c = lane; c < 2 * D; c += 64) {
            Sum<T> v = shares[wave][c / D][c % D];
#pragma unroll
            for (int h = 0; h < Lane<T, D>::kHeads; ++h) v += parts[wave][h][c / D][c % D];
            shares[wave][c / D][c % D] = v;
        }
        wave_lds_sync();
    };
    int rows = 0;                      // in a lane's sums
    if (NORM && kRows<T>)
#pragma unroll
        for (int c = lane; c < 2 * D; c += 64) shares[wave][c / D][c % D] = 0;
    const int64_t units = (int64_t)p.batch * p.tokens * p.parts;
    const int q_groups = (p.heads + me.kHeads - 1) / me.kHeads, k_groups = (p.kv_heads + me.kHeads - 1) / me.kHeads;
    Pair<T> weights[2];
    if (NORM) {
        weights[0].load(static_cast<const T *>(p.q_weight) + me.a, static_cast<const T *>(p.q_weight) + me.b);
        weights[1].load(static_cast<const T *>(p.k_weight) + me.a, static_cast<const T *>(p.k_weight) + me.b);
    }
    for (int64_t unit = (int64_t)blockIdx.x * kWaves + wave; unit < units; unit += (int64_t)gridDim.x * kWaves) {
        const int64_t token = unit / p.parts;
        const int part = (int)(unit - token * p.parts), b = (int)(token / p.tokens), i = (int)(token - (int64_t)b * p.tokens);
        const int q_len = p.q_lengths ? min(max(p.q_lengths[b], 0), p.tokens) : p.tokens;
        const bool there = i < q_len;
        bool angles = false;
        auto side = [&](const void *data, const Strides &s, const void *dout, const Strides &ds, void *out, int heads, int from, int groups, auto which) {
            constexpr int K = decltype(which)::value;
            const T *src = static_cast<const T *>(data) + b * s.batch + (int64_t)i * s.row;
            const T *up = static_cast<const T *>(dout) + b * ds.batch + (int64_t)i * ds.row;
            Pair<T> x_next, g_next;
            auto fetch = [&](int group) {
                const int h = group * me.kHeads + me.slot;
                if (!there || h >= heads) return;
                g_next.load(up + h * ds.head + me.a, up + h * ds.head + me.b);
                if (NORM) x_next.load(src + h * s.head + me.a, src + h * s.head + me.b);
            };
            if (from < groups) fetch(from);
            if (there && !angles) make_angles(p, b, i, q_len, lane, table[wave]);
            angles = true;
            for (int group = from; group < groups; group += p.parts) {
                const int h = group * me.kHeads + me.slot;
                float ga[E], gb[E], x[E], y[E];
                g_next.widen(ga, gb);
                if (NORM) x_next.widen(x, y);
                if (group + p.parts < groups) fetch(group + p.parts);
                if (there && h < heads) {
                    float2 cs[E];
                    own_angles<T, D>(me, table[wave], cs);
                    turn<T, D>(p, me, cs, -1.f, ga, gb);
                    if (NORM) {
                        float by, wa[E], wb[E], dot = 0.f;
                        const float r = inverse_rms<T, D>(x, y, p.eps, &by);
                        weights[K].widen(wa, wb);
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            x[e] *= r; y[e] *= r;
                            sum[K][0][e] += ga[e] * x[e];
                            sum[K][1][e] += gb[e] * y[e];
                            ga[e] *= wa[e]; gb[e] *= wb[e];
                            dot += ga[e] * x[e] + gb[e] * y[e];
                        }
                        dot = lanes_sum<Lane<T, D>::kLanes>(dot) * (1.f / D);
#pragma unroll
                        for (int e = 0; e < E; ++e) { ga[e] = (ga[e] - x[e] * dot) * r * by; gb[e] = (gb[e] - y[e] * dot) * r * by; }
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < E; ++e) ga[e] = gb[e] = 0.f;
                }
                if (h >= heads) continue;
                T *dst = static_cast<T *>(out) + (token * heads + h) * D;
                put(dst + me.a, ga);
                put(dst + me.b, gb);
            }
        };
        // group n of queries and keys together is part n modulo the parts'
        side(p.q, p.qs, grads.dq_out, grads.dqs, grads.dq, p.heads, part, q_groups, std::integral_constant<int, 0>{});
        side(p.k, p.ks, grads.dk_out, grads.dks, grads.dk, p.kv_heads, (part + p.parts - q_groups % p.parts) % p.parts, k_groups, std::integral_constant<int, 1>{});
        if constexpr (NORM && kRows<T>)
            if ((rows += (q_groups + k_groups + p.parts - 1) / p.parts) >= kRows<T>) {
                collect();
                rows = 0;
            }
    }
    if (!NORM) return;
    // over the wavefront's heads, then its workgroup's wavefronts
    if constexpr (kRows<T> != 0) {
        collect();
    } else {
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    float v = sum[k][h][e];
                    for (int d = Lane<T, D>::kLanes; d < 64; d <<= 1) v += __shfl_xor(v, d);
                    if (me.slot == 0) shares[wave][k][(h ? me.b : me.a) + e] = v;
                }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * D; c += kThreads) {
        Sum<T> v = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) v += shares[w][c / D][c % D];
        grads.sums[(int64_t)blockIdx.x * 2 * D + c] = (float)v;
    }
}

// dw in 64 bits: four columns a workgroup, a thread for every so many rows.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void weights_kernel(const float *sums, int rows, T *dq_weight, T *dk_weight) {
    __shared__ double part[kWaves][4];
    const int lane = threadIdx.x & 63, c = blockIdx.x * 4;
    double v[4] = {0.0, 0.0, 0.0, 0.0};
    for (int r = threadIdx.x; r < rows; r += kThreads) {
        const float4 x = *reinterpret_cast<const float4 *>(sums + (int64_t)r * 2 * D + c);
        v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += __shfl_xor(v[i], d);
    if (lane == 0)
#pragma unroll
        for (int i = 0; i < 4; ++i) part[threadIdx.x >> 6][i] = v[i];
    __syncthreads();
    if (threadIdx.x >= 4) return;
    double total = 0.0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) total += part[w][threadIdx.x];
    const int at = c + (int)threadIdx.x;
    (at < D ? dq_weight : dk_weight)[at % D] = (T)(float)total;
}

constexpr const char *kWhat = "rotation";

int problem_of(const fg_rotate_args *a, Problem *p) {
    if (!a) return fail(FG_ERR_ARG, "rotation: arguments are a null pointer");
    if (a->type != FG_TYPE_F32 && a->type != FG_TYPE_F16 && a->type != FG_TYPE_BF16) return fail(FG_ERR_ARG, "rotation: unknown type %d", a->type);
    if (a->batch < 0 || a->tokens < 0 || a->heads < 1 || a->kv_heads < 1) return fail(FG_ERR_ARG, "rotation: negative sizes, or no heads");
    if (a->head_len != 32 && a->head_len != 64 && a->head_len != 128) return fail(FG_ERR_SHAPE, "rotation: heads of 32, 64 or 128 elements, got %d", a->head_len);
    if (a->rotary_len < 0 || a->rotary_len > a->head_len || a->rotary_len % 16)
        return fail(FG_ERR_SHAPE, "rotation: a multiple of 16 elements of a head of %d can be turned, got %d", a->head_len, a->rotary_len);
    if (!(a->eps >= 0.f)) return fail(FG_ERR_ARG, "rotation: eps has to be 0 or more");
    if (a->tokens > (1 << 30) || a->heads > (1 << 20) || a->kv_heads > (1 << 20)) return fail(FG_ERR_SHAPE, "rotation: more than 2^30 tokens or 2^20 heads");
    if (a->axes < 1 || a->axes > 8 || (a->axes > 1 && a->rotary_len && !a->positions))
        return fail(FG_ERR_ARG, "rotation: 1 to 8 axes, and positions with more than one, got %d", a->axes);
    *p = Problem{};
    for (int i = 0; i < a->rotary_len / 2; ++i) {
        if (a->axis[i] >= a->axes) return fail(FG_ERR_ARG, "rotation: pair %d turns by axis %d of %d", i, a->axis[i], a->axes);
        p->turns[i] = a->turns[i];
        p->axis[i] = a->axis[i];
    }
    if ((!a->q_weight) != (!a->k_weight)) return fail(FG_ERR_ARG, "rotation: weights for queries and keys come together");
    const int size = a->type == FG_TYPE_F32 ? 4 : 2;
    int rc;
    if ((rc = block::strides_of("q", a->q, a->q_strides, size, &p->qs, kWhat)) || (rc = block::strides_of("k", a->k, a->k_strides, size, &p->ks, kWhat)) ||
        (rc = block::aligned("the queries' weights", a->q_weight, 16, kWhat)) || (rc = block::aligned("the keys' weights", a->k_weight, 16, kWhat)) ||
        (rc = block::aligned("positions", a->positions, 4, kWhat)) || (rc = block::aligned("lengths", a->lengths, 4, kWhat)) ||
        (rc = block::aligned("q_lengths", a->q_lengths, 4, kWhat)) || (rc = block::aligned("the turned queries", a->q_out, 16, kWhat)) ||
        (rc = block::aligned("the turned keys", a->k_out, 16, kWhat))) return rc;
    p->batch = a->batch; p->tokens = a->tokens; p->heads = a->heads; p->kv_heads = a->kv_heads;
    p->rotary_len = a->rotary_len; p->interleaved = a->interleaved != 0; p->axes = a->axes; p->eps = a->eps;
    p->q = a->q; p->k = a->k; p->q_weight = a->q_weight; p->k_weight = a->k_weight;
    p->positions = a->positions; p->lengths = a->lengths; p->q_lengths = a->q_lengths;
    // A wavefront takes all groups of a token's heads, for which it makes the angles once, or one of them where tokens alone would not fill the card.
    // One wavefront a token / one a group, forward and gradients (us): 32 / 8 heads of 128 in bfloat16 256 tokens 6.9 and 13.8 / 3.9 and 11.1, 1,024 8.0 and 15.6 /
    // 6.3 and 15.9, 2,048 10.4 and 19.9 / 10.4 and 21.3, 4,096 15.3 and 25.8 / 17.0 and 29.6; 6 / 2 of 64 in 32 bits 1,024 4.1 and 9.0 / 3.6 and 9.2, 2,048
    // 4.7 and 10.2 / 4.7 and 11.7, 8,192 9.1 and 18.3 / 10.7 and 20.8.
    const int lanes = a->head_len / 2 / (16 / size), each = 64 / lanes;
    const int groups = (a->heads + each - 1) / each + (a->kv_heads + each - 1) / each;
    p->parts = (int64_t)a->batch * a->tokens >= 2048 ? 1 : groups;
    const int64_t grid = ((int64_t)a->batch * a->tokens * p->parts + kWaves - 1) / kWaves;
    if (grid > block::kMostGroups) return fail(FG_ERR_SHAPE, "rotation: %lld workgroups do not fit a launch", (long long)grid);
    return FG_OK;
}

// Workgroups of the gradients: as many as the card holds at a time, which go on from token to token.
int backward_grid(const Problem &p, const fg_rotate_args *a) {
    const int64_t most = 256 * (a->q_weight && a->type != FG_TYPE_F32 ? kResident<__bf16, true> : kResident<float, true>);
    return (int)std::min(most, ((int64_t)p.batch * p.tokens * p.parts + kWaves - 1) / kWaves);
}

template <typename F> int by_shape(const fg_rotate_args *a, F f) {
    auto with_norm = [&](auto t, auto d) { return a->q_weight ? f(t, d, std::true_type{}) : f(t, d, std::false_type{}); };
    auto with_length = [&](auto t) {
        switch (a->head_len) {
        case 32: return with_norm(t, std::integral_constant<int, 32>{});
        case 64: return with_norm(t, std::integral_constant<int, 64>{});
        default: return with_norm(t, std::integral_constant<int, 128>{});
        }
    };
    switch (a->type) {
    case FG_TYPE_F32: return with_length(float{});
    case FG_TYPE_F16: return with_length(_Float16{});
    default: return with_length(__bf16{});
    }
}

}  // namespace
}  // namespace rotate
}  // namespace fg

extern "C" int fg_rotate_heads(const fg_rotate_args *args, void *stream) {
    using namespace fg;
    using namespace fg::rotate;
    Problem p;
    if (int rc = problem_of(args, &p)) return rc;
    if ((int64_t)p.batch * p.tokens == 0) return FG_OK;
    if (!p.q || !p.k || !args->q_out || !args->k_out) return fail(FG_ERR_ARG, "rotation: null pointer");
    const dim3 grid((unsigned)(((int64_t)p.batch * p.tokens * p.parts + kWaves - 1) / kWaves));
    by_shape(args, [&](auto t, auto d, auto norm) {
        typedef decltype(t) T;
        rotate_kernel<T, decltype(d)::value, decltype(norm)::value><<<grid, dim3(kThreads), 0, static_cast<hipStream_t>(stream)>>>(
            p, static_cast<T *>(args->q_out), static_cast<T *>(args->k_out));
        return 0;
    });
    FG_HIP_TRY(hipGetLastError());
    return FG_OK;
}

extern "C" int64_t fg_rotate_heads_backward_workspace(const fg_rotate_args *args) {
    fg::rotate::Problem p;
    if (int rc = fg::rotate::problem_of(args, &p)) return rc;
    return args->q_weight ? (int64_t)fg::rotate::backward_grid(p, args) * 2 * args->head_len * (int64_t)sizeof(float) : 0;
}

extern "C" int fg_rotate_heads_backward(const fg_rotate_args *args, const fg_rotate_grads *grads, void *workspace, size_t workspace_bytes, void *stream) {
    using namespace fg;
    using namespace fg::rotate;
    Problem p;
    int rc;
    if ((rc = problem_of(args, &p))) return rc;
    if (!grads) return fail(FG_ERR_ARG, "rotation: gradients are a null pointer");
    const int size = args->type == FG_TYPE_F32 ? 4 : 2;
    Grads g{grads->dq_out, grads->dk_out, {}, {}, grads->dq, grads->dk, static_cast<float *>(workspace)};
    if ((rc = block::strides_of("dL/d(turned queries)", grads->dq_out, grads->dq_out_strides, size, &g.dqs, kWhat)) ||
        (rc = block::strides_of("dL/d(turned keys)", grads->dk_out, grads->dk_out_strides, size, &g.dks, kWhat)) ||
        (rc = block::aligned("dq", grads->dq, 16, kWhat)) || (rc = block::aligned("dk", grads->dk, 16, kWhat)) ||
        (rc = block::aligned("the weights' gradients", grads->dq_weight, size, kWhat)) ||
        (rc = block::aligned("the weights' gradients", grads->dk_weight, size, kWhat)) || (rc = block::aligned("the workspace", workspace, 16, kWhat))) return rc;
    const bool norm = args->q_weight;
    if (norm && (!grads->dq_weight || !grads->dk_weight)) return fail(FG_ERR_ARG, "rotation: null pointer");
    const int rows = backward_grid(p, args);
    const size_t need = norm ? (size_t)rows * 2 * args->head_len * sizeof(float) : 0;
    if (workspace_bytes < need || (need && !workspace))
        return fail(FG_ERR_ARG, "rotation: a workspace of %zu bytes, %zu needed (fg_rotate_heads_backward_workspace)", workspace_bytes, need);
    if (rows && (!grads->dq_out || !grads->dk_out || !grads->dq || !grads->dk || (norm && (!p.q || !p.k)))) return fail(FG_ERR_ARG, "rotation: null pointer");
    hipStream_t s = static_cast<hipStream_t>(stream);
    rc = by_shape(args, [&](auto t, auto d, auto with_norm) -> int {
        typedef decltype(t) T;
        constexpr int D = decltype(d)::value;
        constexpr bool NORM = decltype(with_norm)::value;
        if (rows) rotate_backward_kernel<T, D, NORM><<<dim3((unsigned)rows), dim3(kThreads), 0, s>>>(p, g);
        FG_HIP_TRY(hipGetLastError());
        if (NORM) weights_kernel<T, D><<<dim3(2 * D / 4), dim3(kThreads), 0, s>>>(g.sums, rows, static_cast<T *>(grads->dq_weight), static_cast<T *>(grads->dk_weight));
        FG_HIP_TRY(hipGetLastError());
        return FG_OK;
    });
    return rc;
}
