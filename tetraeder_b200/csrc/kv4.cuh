// The 4-bit KV cache: its format, its quantiser, and what the store, decode and prefill kernels share.
//
// A row (sequence, KV head, position) of K or of V is head_dim values in blocks of 32.  A block holds
// d * (c - 8): d one f16 scale, c 4-bit codes (the values of ggml's Q4_0).  Two planes per K and per V:
//   codes  u8  [n_seq][n_kv][n_ctx][head_dim / 2]   value 2j of a block in the low half of its byte j
//   scales f16 [n_seq][n_kv][n_ctx][head_dim / 32]
// A head's rows follow one another, so a tile of positions is one contiguous run of either plane and
// comes into shared memory by one flat bulk copy.  There eight rows are read at a time by ldmatrix, 16
// bytes (one block) each; rows of 64 (32) bytes would put them on 4 (2) of the 8 bank groups, so block
// b's 16-byte chunk sits at slot b ^ kv4_turn(position) of its row: every such read is conflict-free.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include "common.cuh"

namespace tmoe {

struct Kv4Planes {
    uint8_t *kc;
    __half *ks;
    uint8_t *vc;
    __half *vs;
    int n_seq, n_kv, n_ctx;  // n_ctx: positions held per sequence and head, a multiple of 64
};

template <int HD>
__host__ __device__ __forceinline__ int kv4_turn(int pos) {
    return HD == 128 ? (pos >> 1) & 3 : (pos >> 2) & 1;
}

// The cache holds finite values only: a NaN counts as 0, an infinity as the largest float (which the
// scale's own clamp then limits), so that no row can spoil another's products where it is masked.
__device__ __forceinline__ float kv4_finite(float x) {
    return x != x ? 0.0f : fminf(fmaxf(x, -FLT_MAX), FLT_MAX);
}

// From a block's largest and smallest value: its f16 scale d = m / -8, m the value of the largest
// magnitude (the positive one of a pair), and the f32 factor that takes values to codes.
__device__ __forceinline__ void kv4_scale(float hi, float lo, __half &d16, float &inv) {
    const float m = hi >= -lo ? hi : lo;
    const float d = fminf(fmaxf(__fmul_rn(m, -0.125f), -65504.0f), 65504.0f);
    d16 = __float2half_rn(d);
    inv = (__half_as_ushort(d16) & 0x7fffu) == 0 ? 0.0f : __fdiv_rn(1.0f, d);
}
// floor(x inv + 8.5) within 0 .. 15 in the low bits of a float of 2^23's exponent: adding 2^23 downwards leaves the
// floor there, at full rate, where the conversion and floor instructions run at a quarter of it.
__device__ __forceinline__ uint32_t kv4_code_bits(float x, float inv) {
    const float t = fminf(fmaxf(__fadd_rn(__fmul_rn(x, inv), 8.5f), 0.0f), 15.5f);
    return __float_as_uint(__fadd_rd(t, 8388608.0f));
}
// The codes of N <= 8 values as a word, the first in the low bits
template <int N>
__device__ __forceinline__ uint32_t kv4_word(const float *x, float inv) {
    uint32_t w = 0, base = 0;
#pragma unroll
    for (int i = 0; i < N; i++) w += kv4_code_bits(x[i], inv) << (4 * i), base += 0x4b000000u << (4 * i);
    return w - base;
}

// N consecutive activations as f32 (N a multiple of 4; 16-byte aligned, or 8 for four bf16).
template <int N>
__device__ __forceinline__ void kv4_load_row(const float *p, float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        const float4 a = __ldg(reinterpret_cast<const float4 *>(p + i));
        v[i] = a.x, v[i + 1] = a.y, v[i + 2] = a.z, v[i + 3] = a.w;
    }
}
__device__ __forceinline__ void kv4_bf2(uint32_t u, float &a, float &b) {
    a = __uint_as_float(u << 16), b = __uint_as_float(u & 0xffff0000u);
}
template <int N>
__device__ __forceinline__ void kv4_load_row(const __nv_bfloat16 *p, float (&v)[N]) {
    if constexpr (N % 8 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 8) {
            const uint4 a = __ldg(reinterpret_cast<const uint4 *>(p + i));
            kv4_bf2(a.x, v[i], v[i + 1]), kv4_bf2(a.y, v[i + 2], v[i + 3]);
            kv4_bf2(a.z, v[i + 4], v[i + 5]), kv4_bf2(a.w, v[i + 6], v[i + 7]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint2 a = __ldg(reinterpret_cast<const uint2 *>(p + i));
            kv4_bf2(a.x, v[i], v[i + 1]), kv4_bf2(a.y, v[i + 2], v[i + 3]);
        }
    }
}
__device__ __forceinline__ uint32_t kv4_pack_bf2(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    uint32_t u;
    memcpy(&u, &h, 4);
    return u;
}
// N consecutive values to activations (N a multiple of 8).
template <int N>
__device__ __forceinline__ void kv4_store_row(float *p, const float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 4) *reinterpret_cast<float4 *>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
}
template <int N>
__device__ __forceinline__ void kv4_store_row(__nv_bfloat16 *p, const float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 8)
        *reinterpret_cast<uint4 *>(p + i) = make_uint4(kv4_pack_bf2(v[i], v[i + 1]), kv4_pack_bf2(v[i + 2], v[i + 3]),
                                                       kv4_pack_bf2(v[i + 4], v[i + 5]), kv4_pack_bf2(v[i + 6], v[i + 7]));
}

__device__ __forceinline__ uint32_t kv4_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    uint32_t u;
    memcpy(&u, &h, 4);
    return u;
}
// 2^e, e in [-126, 127]
__device__ __forceinline__ float kv4_pow2(int e) { return __int_as_float((127 + e) << 23); }
// 1 / p, p = 2^e for e in [-126, 126]
__device__ __forceinline__ float kv4_inv_pow2(float p) { return __uint_as_float(0x7f000000u - __float_as_uint(p)); }
__device__ __forceinline__ float kv4_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A row's factor from S to log2 scores, within a float's range: not 0, as masked scores are -inf times it, and not infinite, as
// a score of 0 is 0 times it.  Queries so small have equal scores either way, and ones so large the largest score alone.
__device__ __forceinline__ float kv4_factor(float c) { return fminf(fmaxf(c, FLT_MIN), FLT_MAX); }

// An exponent is s c - ref in one multiply-add, ref the rounded s c of a row's largest score s.  From |ref| = 2^24 on, what that
// rounding left would be an exponent of its own, past a float's in the end.  There c and ref are held below, times
// 2^-kv4_far(ref): scores whose difference a float can tell at all still differ by more than a weight's bits, or by less than
// the scores' own error.
__device__ __forceinline__ int kv4_far(float ref) {
    const int e = (int)((__float_as_uint(ref) >> 23) & 255u) - 127;
    return e >= 24 && e < 128 ? e - 23 : 0;
}

// The attention calls' scratch: counters (zero between calls), then the parts of split work.
inline size_t kv4_counter_bytes(int sm_count) { return ((size_t)sm_count * 8 + 15) / 16 * 16; }
inline float *kv4_scratch_parts(void *scratch, int sm_count) {
    return reinterpret_cast<float *>(static_cast<char *>(scratch) + kv4_counter_bytes(sm_count));
}

// Which positions a query at position `last` sees: those up to it, of them (window > 0) the last
// `window` and the first n_sink.  As TILE-position tiles: the sinks' tiles 0 .. head - 1, then those
// from `body` on.
struct Kv4Seen {
    int len;   // positions 0 .. len - 1 exist
    int from;  // the window's first position
    int head, body, tiles;
    template <int TILE>
    static __host__ __device__ __forceinline__ Kv4Seen of(int last, int window, int n_sink) {
        Kv4Seen s;
        s.len = last + 1;
        s.from = window > 0 && s.len > window ? s.len - window : 0;
        const int sinks = n_sink < s.from ? n_sink : s.from;
        s.head = (sinks + TILE - 1) / TILE;
        s.body = s.from / TILE > s.head ? s.from / TILE : s.head;
        s.tiles = s.head + (s.len + TILE - 1) / TILE - s.body;
        return s;
    }
    __device__ __forceinline__ int tile(int i) const { return i < head ? i : body + (i - head); }
    __device__ __forceinline__ bool sees(int p, int n_sink) const { return p < len && (p >= from || p < n_sink); }
    // whether all of positions p .. p + n - 1 are seen
    __device__ __forceinline__ bool whole(int p, int n, int n_sink) const {
        return p + n <= len && (p >= from || p + n <= n_sink);
    }
};

}  // namespace tmoe
