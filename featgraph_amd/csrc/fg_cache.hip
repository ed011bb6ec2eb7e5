// Keys and values into a cache of 4 or 8 bits, and back.
//   write:  for 32 neighbouring elements x of a head  e = the least power with which max |x| 2^-e rounds to at most the largest element (6 of e2m1,
//           448 of e4m3), -127 <= e; codes = x 2^-e to the nearest element, ties to the even code.  A power of two divides without rounding, so that
//           codes are the same on every machine that follows the rule.
//   read:   code 2^e, rounded to the type (float16: and no further than its largest number, for an element may be larger than the value it came from).
//
// What bounds them.  16,384 tokens of 8 heads of 128, K and V, bfloat16 and 4 bits (86 MB): written in 17.5 us, 4.9 TB/s, the rate of a large copy; read in
// 14.2 us (6.0 TB/s, part of it from the Infinity Cache). One token each of 32 sequences 3.3 us, a launch.
#include <algorithm>
#include <limits>

#include "fg_cache.h"

namespace fg {
namespace cache {

namespace {

using block::Strides;
using block::V8;
using block::load8;

constexpr int kThreads = 256;

struct Window {                        // tokens of a call and where they stand in the cache
    int batch, tokens, keys, kv_heads;
    const int32_t *lengths, *q_lengths, *first;
    int lanes_shift, parts;            // see Places
};

// A thread takes kEach times eight elements of one head of K or V.  The D / 8 of a token follow one another, then the tokens of the head: codes are
// written, and read, as whole lines.  2^lanes_shift threads share one of `parts` parts of a head, the others of a workgroup take other heads, so that an
// index is divided once a thread (with divisions for every eight elements, and these alone a thread's, 16,384 tokens of 8 x 128 are written in 21.8 us and read in 20.5).
constexpr int kEach = 4;
template <int D> struct Places {
    static constexpr int C = D / 8;
    bool second, there;                // V; any work
    int b, g, at, step, col;           // at, at + step ..: of the head's pieces; `step` is a multiple of C or there is one piece only
    int64_t row;                       // of (batch, kv_heads)
    __device__ __forceinline__ Places(const Window &w) {
        const unsigned half = gridDim.x >> 1, block = blockIdx.x >= half ? blockIdx.x - half : blockIdx.x;
        second = blockIdx.x >= half;
        const unsigned group = block / w.parts, part = block - group * w.parts;
        step = 1 << w.lanes_shift;
        row = (int64_t)group * (kThreads >> w.lanes_shift) + (threadIdx.x >> w.lanes_shift);
        there = row < (int64_t)w.batch * w.kv_heads;
        b = (int)((unsigned)row / (unsigned)w.kv_heads);
        g = (int)(row - (int64_t)b * w.kv_heads);
        at = (int)part * step * kEach + (threadIdx.x & (step - 1));
        col = at % C * 8;
    }
    __device__ __forceinline__ int token(int u) const { return (at + u * step) / C; }
};

// The larger of two lanes' numbers, over four neighbouring lanes.
__device__ __forceinline__ unsigned quad_max(unsigned v) {
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true));      // quad_perm [1,0,3,2]
    return max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true));   // quad_perm [2,3,0,1]
}

struct Source { const void *data; Strides s; void *codes, *scales; };

// Eight numbers' codes, and the byte of the scale that the lane's four neighbours share.
template <int BITS> __device__ __forceinline__ unsigned codes_of(const float (&f)[8], uint32_t (&word)[BITS / 4]) {
    unsigned most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(f[i]) & 0x7fffffffu);       // as numbers are ordered; infinities and NaN above them
    most = quad_max(most);
    // max |x| = 2^(high - 127) (1 + low / 2^23); 1.75 and more (e2m1) and what is above 1.8125 (e4m3) would round to the next power of two
    const int high = (int)(most >> 23), low = (int)(most & 0x7fffffu);
    const int up = BITS == 4 ? low >= 0x600000 : low > 0x680000;
    const int byte = min(max(high - (BITS == 4 ? 2 : 8) + up, 0), kTopExponent<BITS> + 127);
    const float scale = scale_of((unsigned)byte);
    if constexpr (BITS == 4) {
        uint32_t c = 0;
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[0], f[1], scale, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[2], f[3], scale, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[4], f[5], scale, 2);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[6], f[7], scale, 3);
        word[0] = c;
    } else {
        // the conversion makes NaN of what is beyond the largest element, which the scale's own limit allows: 448 2^119 at most
        constexpr float TOP = 0x1.cp127f;
        typedef short s16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = fminf(fmaxf(f[4 * h + i], -TOP), TOP);
            s16x2 c = {0, 0};
            c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, y[0], y[1], scale, false);
            c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, y[2], y[3], scale, true);
            word[h] = __builtin_bit_cast(uint32_t, c);
        }
    }
    if (most < 0x7f800000u) return (unsigned)byte;
#pragma unroll
    for (int i = 0; i < BITS / 4; ++i) word[i] = 0;
    return 255;
}

template <typename T, int D, int BITS>
__global__ __launch_bounds__(kThreads) void write_kernel(const Window w, const Source ks, const Source vs) {
    const Places<D> p(w);
    if (!p.there) return;              // the lanes of one scale stay together: a head's pieces are a multiple of four
    const Source &s = p.second ? vs : ks;
    const int q_len = w.q_lengths ? min(max(w.q_lengths[p.b], 0), w.tokens) : w.tokens;
    const int k_len = w.lengths ? min(max(w.lengths[p.b], 0), w.keys) : w.keys;
    const T *src = static_cast<const T *>(s.data) + p.b * s.s.batch + p.g * s.s.head + p.col;
    V8<T> x[kEach];
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
        const int i = p.token(u);
        if (i < q_len && k_len - q_len + i >= 0) x[u] = load8(src + (int64_t)i * s.s.row);
    }
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
        const int i = p.token(u), key = k_len - q_len + i;
        if (i >= q_len || key < 0) continue;
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = (float)x[u][e];
        uint32_t word[BITS / 4];
        const unsigned byte = codes_of<BITS>(f, word);
        const int64_t row = p.row * w.keys + key;
        uint8_t *out = static_cast<uint8_t *>(s.codes) + row * (D * BITS / 8) + p.col * BITS / 8;
        if constexpr (BITS == 4) *reinterpret_cast<uint32_t *>(out) = word[0];
        else *reinterpret_cast<uint2 *>(out) = make_uint2(word[0], word[1]);
        if (p.col % kGroup == 0) static_cast<uint8_t *>(s.scales)[row * (D / kGroup) + p.col / kGroup] = (uint8_t)byte;
    }
}

struct Target { const void *codes, *scales; void *out; };

template <typename T, int D, int BITS>
__global__ __launch_bounds__(kThreads) void read_kernel(const Window w, const Target kt, const Target vt) {
    const Places<D> p(w);
    if (!p.there) return;
    const Target &t = p.second ? vt : kt;
    const int k_len = w.lengths ? min(max(w.lengths[p.b], 0), w.keys) : w.keys;
    const int64_t first = w.first ? w.first[p.b] : 0;
    uint32_t word[kEach][BITS / 4];
    unsigned byte[kEach];
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
        const int64_t key = first + p.token(u);
        if (p.token(u) < w.tokens && key >= 0 && key < k_len) {
            const int64_t row = p.row * w.keys + key;
            const uint8_t *src = static_cast<const uint8_t *>(t.codes) + row * (D * BITS / 8) + p.col * BITS / 8;
            if constexpr (BITS == 4) {
                word[u][0] = *reinterpret_cast<const uint32_t *>(src);
            } else {
                const uint2 two = *reinterpret_cast<const uint2 *>(src);
                word[u][0] = two.x; word[u][1] = two.y;
            }
            byte[u] = static_cast<const uint8_t *>(t.scales)[row * (D / kGroup) + p.col / kGroup];
        }
    }
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
        const int i = p.token(u);
        const int64_t key = first + i;
        if (i >= w.tokens) continue;
        V8<T> x = block::zero8<T>();
        if (key >= 0 && key < k_len) {
            const auto y = values<BITS, typename std::conditional<sizeof(T) == 4, float, __bf16>::type>(word[u], scale_of(byte[u]));
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = (T)within<T>((float)y[e]);
        }
        *reinterpret_cast<V8<T> *>(static_cast<T *>(t.out) + (((int64_t)p.b * w.tokens + i) * w.kv_heads + p.g) * D + p.col) = x;
    }
}

template <typename F> int by_shape(int type, int head_len, int bits, F f) {
    auto with_bits = [&](auto t, auto d) {
        return bits == 4 ? f(t, d, std::integral_constant<int, 4>{}) : f(t, d, std::integral_constant<int, 8>{});
    };
    auto with_length = [&](auto t) {
        switch (head_len) {
        case 32: return with_bits(t, std::integral_constant<int, 32>{});
        case 64: return with_bits(t, std::integral_constant<int, 64>{});
        default: return with_bits(t, std::integral_constant<int, 128>{});
        }
    };
    switch (type) {
    case FG_TYPE_F32: return with_length(float{});
    case FG_TYPE_F16: return with_length(_Float16{});
    default: return with_length(__bf16{});
    }
}

// How the tokens' pieces are dealt out, and the workgroups for that.
int cut(Window *w, int head_len, unsigned *grid) {
    const int64_t pieces = (int64_t)w->tokens * (head_len / 8), rows = (int64_t)w->batch * w->kv_heads;
    w->lanes_shift = 0;
    while ((1 << w->lanes_shift) < kThreads && (1 << w->lanes_shift) < pieces) ++w->lanes_shift;
    const int64_t lanes = 1 << w->lanes_shift, heads = kThreads >> w->lanes_shift, parts = (pieces + lanes * kEach - 1) / (lanes * kEach);
    const int64_t n = 2 * ((rows + heads - 1) / heads) * parts;
    if (pieces > INT32_MAX - kThreads * kEach || rows > INT32_MAX || n > block::kMostGroups) return fail(FG_ERR_SHAPE, "cache: %lld workgroups do not fit a launch", (long long)n);
    w->parts = (int)parts;
    *grid = (unsigned)n;
    return FG_OK;
}

int known(int type) {
    return type == FG_TYPE_F32 || type == FG_TYPE_F16 || type == FG_TYPE_BF16 ? FG_OK : fail(FG_ERR_ARG, "cache: unknown type %d", type);
}

}  // namespace

int check(const fg_kv_cache *c) {
    if (!c) return fail(FG_ERR_ARG, "cache: null pointer");
    if (c->bits != 4 && c->bits != 8) return fail(FG_ERR_ARG, "cache: elements of 4 or 8 bits, got %d", c->bits);
    if (c->batch < 0 || c->keys < 0 || c->kv_heads < 1) return fail(FG_ERR_ARG, "cache: negative sizes, or no heads");
    if (c->head_len != 32 && c->head_len != 64 && c->head_len != 128) return fail(FG_ERR_SHAPE, "cache: heads of 32, 64 or 128 elements, got %d", c->head_len);
    if (c->keys > (1 << 30)) return fail(FG_ERR_SHAPE, "cache: more than 2^30 keys");
    const bool any = (int64_t)c->batch * c->keys;
    if (any && (!c->k || !c->v || !c->k_scales || !c->v_scales)) return fail(FG_ERR_ARG, "cache: null pointer");
    if (reinterpret_cast<uintptr_t>(c->k) % 16 || reinterpret_cast<uintptr_t>(c->v) % 16 || reinterpret_cast<uintptr_t>(c->k_scales) % 4 ||
        reinterpret_cast<uintptr_t>(c->v_scales) % 4)
        return fail(FG_ERR_ARG, "cache: codes have to stand at multiples of 16 bytes, scales of 4 bytes");
    return FG_OK;
}

}  // namespace cache
}  // namespace fg

extern "C" int fg_cache_write(const fg_kv_cache *cache, int type, const void *k_dev, const int64_t *k_strides, const void *v_dev, const int64_t *v_strides,
                              int tokens, const int32_t *lengths_dev, const int32_t *q_lengths_dev, void *stream) {
    using namespace fg;
    using namespace fg::cache;
    int rc;
    if ((rc = cache::check(cache)) || (rc = known(type))) return rc;
    if (tokens < 0 || tokens > (1 << 30)) return fail(FG_ERR_ARG, "cache: %d new tokens", tokens);
    if (!k_strides || !v_strides) return fail(FG_ERR_ARG, "cache: null pointer");
    const int size = type == FG_TYPE_F32 ? 4 : 2;
    Source ks{k_dev, {}, cache->k, cache->k_scales}, vs{v_dev, {}, cache->v, cache->v_scales};
    if ((rc = block::strides_of("k", k_dev, k_strides, size, &ks.s, "cache")) || (rc = block::strides_of("v", v_dev, v_strides, size, &vs.s, "cache")) ||
        (rc = block::aligned("lengths", lengths_dev, 4, "cache")) || (rc = block::aligned("q_lengths", q_lengths_dev, 4, "cache"))) return rc;
    if ((int64_t)cache->batch * tokens == 0 || cache->keys == 0) return FG_OK;
    if (!k_dev || !v_dev) return fail(FG_ERR_ARG, "cache: null pointer");
    Window w{cache->batch, tokens, cache->keys, cache->kv_heads, lengths_dev, q_lengths_dev, nullptr, 0, 0};
    unsigned grid;
    if ((rc = cut(&w, cache->head_len, &grid))) return rc;
    by_shape(type, cache->head_len, cache->bits, [&](auto t, auto d, auto bits) {
        write_kernel<decltype(t), decltype(d)::value, decltype(bits)::value><<<dim3(grid), dim3(kThreads), 0, static_cast<hipStream_t>(stream)>>>(w, ks, vs);
        return 0;
    });
    FG_HIP_TRY(hipGetLastError());
    return FG_OK;
}

extern "C" int fg_cache_read(const fg_kv_cache *cache, int type, void *k_dev, void *v_dev, int count, const int32_t *first_dev, const int32_t *lengths_dev,
                             void *stream) {
    using namespace fg;
    using namespace fg::cache;
    int rc;
    if ((rc = cache::check(cache)) || (rc = known(type))) return rc;
    if (count < 0 || count > (1 << 30)) return fail(FG_ERR_ARG, "cache: %d keys to read", count);
    if ((rc = block::aligned("k", k_dev, 16, "cache")) || (rc = block::aligned("v", v_dev, 16, "cache")) || (rc = block::aligned("first", first_dev, 4, "cache")) ||
        (rc = block::aligned("lengths", lengths_dev, 4, "cache"))) return rc;
    if ((int64_t)cache->batch * count == 0) return FG_OK;
    if (!k_dev || !v_dev) return fail(FG_ERR_ARG, "cache: null pointer");
    Window w{cache->batch, count, cache->keys, cache->kv_heads, lengths_dev, nullptr, first_dev, 0, 0};
    unsigned grid;
    if ((rc = cut(&w, cache->head_len, &grid))) return rc;
    const Target kt{cache->k, cache->k_scales, k_dev}, vt{cache->v, cache->v_scales, v_dev};
    by_shape(type, cache->head_len, cache->bits, [&](auto t, auto d, auto bits) {
        read_kernel<decltype(t), decltype(d)::value, decltype(bits)::value><<<dim3(grid), dim3(kThreads), 0, static_cast<hipStream_t>(stream)>>>(w, kt, vt);
        return 0;
    });
    FG_HIP_TRY(hipGetLastError());
    return FG_OK;
}
