// Attention of many query tokens of one sequence over the 4-bit KV cache (format: kv4.cuh), on the
// 5th-generation tensor cores.
//
// The query rows of a KV head are its tokens times the query heads that share it (row r: token r / G, head
// r % G), so that one dequantised tile of K and V serves all of them.  A CTA takes 256 rows, as two
// 128-row tiles A and B, and walks the 128-position tiles that its tokens see:
//   S = Q K^T   tcgen05, Q and K f16 in shared memory (128-byte swizzle), S f32 in TMEM (128 columns a tile)
//   P           a thread per row: exp2(S c - ref) as f16, back into TMEM over S
//   O += P V    tcgen05, P from TMEM, V f16 in shared memory as it lies (rows are positions: an N-major
//               operand), O f32 in TMEM
// Warps: 0-3 and 4-7 the softmax of A and B, 8-11 dequantise, 12 issues the MMAs, 13 the bulk copies.  While
// the softmax of one tile runs, the tensor cores work on the other.
//
// Bound: per 256 rows x 128 positions of 128-wide heads the MMAs take 2048 clocks and so do the exps (16 a
// clock and SM); the dequantisation (13 instructions for 8 values, about 475 issue slots a scheduler)
// hides beside them.
//   - A code under a mask is 1024 + c in f16; minus 1032, times the block's scale: f16(d (c - 8)).  The pairs that
//     fall out of a word are values (0, 4), (1, 5), (2, 6), (3, 7); Q's chunks are written in that order,
//     and O's columns come out in it.
//   - The running reference of a row moves only when a score exceeds it by more than 2^8: until then P is
//     taken against the old one (below 2^14 in f16, as it starts at 2^6), and O needs no rescaling.  A
//     tile is first tried with the old reference, S still whole in TMEM; the rare failure is redone.
//   - Q is scaled per row by a power of two into f16's range.  Scales are held to what f16 can carry times 8.
//   - Few query rows leave SMs idle, so their positions are split over CTAs, and kv4_join_kernel adds the parts.
#include "kernels.cuh"
#include "kv4.cuh"
#include "tcgen05.cuh"

namespace tmoe {

constexpr int KP_M = 128;            // rows of a tile
constexpr int KP_ROWS = 2 * KP_M;    // of a CTA
constexpr int KP_N = 128;            // positions of a tile
constexpr int KP_WARPS = 14;
constexpr int KP_THREADS = 32 * KP_WARPS;
constexpr int KP_RAW = 3;            // raw tiles (of K or of V) in flight
constexpr float KP_ROOM = 8.0f;      // how far (log2) a score may exceed its row's reference
constexpr float KP_BIAS = 6.0f;      // P is 2^KP_BIAS at the reference
constexpr float KP_SCALE_MAX = 8188.0f;  // 8 * this is f16's largest

struct Kv4PrefillArgs {
    const void *q;
    void *out;
    int64_t q_ld, out_ld;
    int seq, pos0, n_tok, n_head, window, n_sink, splits;
    float scale;
    float *part;  // splits > 1: [cta][KP_ROWS][HD + 2]
    int *err;
};

template <int HD>
struct Kv4PrefillCfg {
    static constexpr int NB = HD / 32, HALVES = HD / 64;  // 64-wide halves of a row: 128 bytes of f16
    static constexpr int HALF = KP_N * 128;               // bytes of a half tile
    static constexpr int TILE = HALVES * HALF;
    static constexpr int CODES = KP_N * HD / 2, SCALES = KP_N * NB * 2, RAW = CODES + SCALES;
    static constexpr int Q = 0, K = 2 * TILE, V = K + 2 * TILE, R = V + 2 * TILE, BARS = R + KP_RAW * RAW;
    static constexpr int SMEM = BARS + 256 + KP_ROWS * 4 + 1024 /* alignment */;
};

struct KpBars {
    uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], raw_full[KP_RAW], raw_empty[KP_RAW], s_full[2],
        p_full[2], o_full[2];
    uint32_t tmem;
};
static_assert(sizeof(KpBars) <= 256, "barrier room");

// Which positions the tokens t0 .. t1 see between them, as tiles of KP_N (see Kv4Seen).
__host__ __device__ __forceinline__ Kv4Seen kp_seen(int pos0, int t0, int t1, int window, int n_sink) {
    Kv4Seen s;
    s.len = pos0 + t1 + 1;
    s.from = window > 0 && pos0 + t0 + 1 > window ? pos0 + t0 + 1 - window : 0;
    const int sinks = n_sink < s.from ? n_sink : s.from;
    s.head = (sinks + KP_N - 1) / KP_N;
    s.body = s.from / KP_N > s.head ? s.from / KP_N : s.head;
    s.tiles = s.head + (s.len + KP_N - 1) / KP_N - s.body;
    return s;
}

// Four f16 pairs d (c - 8) of a word of codes: values (0, 4), (1, 5), (2, 6), (3, 7).
__device__ __forceinline__ uint4 kp_word(uint32_t w, __half2 d) {
    const __half2 off = __float2half2_rn(1032.0f), sixteenth = __float2half2_rn(0.0625f), off16 = __float2half2_rn(-72.0f);
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t u = i & 2 ? w >> 8 : w;
        uint32_t x;
        asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(x) : "r"(u), "r"(i & 1 ? 0x00f000f0u : 0x000f000fu), "r"(0x64006400u));
        __half2 h;
        memcpy(&h, &x, 4);
        h = i & 1 ? __hfma2(h, sixteenth, off16) : __hsub2(h, off);  // both exact
        h = __hmul2(h, d);
        memcpy(&r[i], &h, 4);
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}

// Bounded waits: by one thread, or by a whole warp.  One that runs out latches the error and ends the role.
#define KP_WAIT_WARP(bar, phase)                                                            \
    do {                                                                                    \
        if (!__all_sync(0xffffffffu, mbar_wait_bounded(&(bar), (uint32_t)(phase)))) {       \
            if (lane == 0) latch_error(a.err, TMOE_DEV_ERR_TIMEOUT);                        \
            goto done;                                                                      \
        }                                                                                   \
    } while (0)
#define KP_WAIT(bar, phase)                                  \
    do {                                                     \
        if (!mbar_wait_bounded(&(bar), (uint32_t)(phase))) { \
            latch_error(a.err, TMOE_DEV_ERR_TIMEOUT);        \
            goto done;                                       \
        }                                                    \
    } while (0)

template <int HD, typename T>
__global__ void __launch_bounds__(KP_THREADS, 1) kv4_prefill_kernel(const Kv4PrefillArgs a, const Kv4Planes c) {
    using Cfg = Kv4PrefillCfg<HD>;
    constexpr int NB = Cfg::NB;
    extern __shared__ uint8_t kp_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(kp_raw) + 1023) & ~(uintptr_t)1023);
    KpBars &bars = *reinterpret_cast<KpBars *>(smem + Cfg::BARS);
    float *row_c = reinterpret_cast<float *>(smem + Cfg::BARS + 256);  // [KP_ROWS] log2 score of an accumulator's 1
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // ---- which rows and which tiles; the longest runs (the last tokens) come first
    const int G = a.n_head / c.n_kv, rows = a.n_tok * G, blocks = (rows + KP_ROWS - 1) / KP_ROWS;
    const int sp = blockIdx.x % a.splits, g = (blockIdx.x / a.splits) % c.n_kv;
    const int blk = blocks - 1 - blockIdx.x / (a.splits * c.n_kv);
    const int row0 = blk * KP_ROWS, n_rows = min(KP_ROWS, rows - row0);
    const int mt = n_rows > KP_M ? 2 : 1;
    const Kv4Seen seen = kp_seen(a.pos0, row0 / G, (row0 + n_rows - 1) / G, a.window, a.n_sink);
    const int tile0 = (int)((int64_t)seen.tiles * sp / a.splits), n = (int)((int64_t)seen.tiles * (sp + 1) / a.splits) - tile0;

    if (threadIdx.x == 0) {
        mbar_init(&bars.q_full, 4 * mt);
        for (int i = 0; i < 2; i++) {
            mbar_init(&bars.k_full[i], 4);
            mbar_init(&bars.k_empty[i], 1);
            mbar_init(&bars.v_full[i], 4);
            mbar_init(&bars.v_empty[i], 1);
            mbar_init(&bars.s_full[i], 1);
            mbar_init(&bars.p_full[i], 4);
            mbar_init(&bars.o_full[i], 1);
        }
        for (int i = 0; i < KP_RAW; i++) {
            mbar_init(&bars.raw_full[i], 1);
            mbar_init(&bars.raw_empty[i], 4);
        }
        fence_barrier_init();
    }
    if (warp == 12) tc::alloc(&bars.tmem, 512);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = bars.tmem;
    pdl_wait();
    pdl_trigger();

    if (warp < 8) {
        // ------------------------------------------------------------ Q, then the softmax: a thread per row
        const int m = warp >> 2;
        if (m < mt) {
            // half a warp per row, 8 values a lane
            for (int i = 0; i < 32; i += 32 / (HD / 8)) {
                const int r = (warp & 3) * 32 + i + lane / (HD / 8), ch = lane % (HD / 8);  // row of the tile, chunk
                const int row = row0 + m * KP_M + r;
                float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                if (row < rows)
                    kv4_load_row(reinterpret_cast<const T *>(a.q) + (int64_t)(row / G) * a.q_ld +
                                     (int64_t)(g * G + row % G) * HD + 8 * ch, x);
                float top = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[e]));
#pragma unroll
                for (int o = HD / 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                // 2^e * top in [2^5, 2^6): exact for bf16 values down to 2^-22 of the largest
                const int e = top > 0.0f && top <= FLT_MAX ? 5 - ilogbf(top) : 0;
                const int e1 = e / 2, e2 = e - e1;
                const float up1 = kv4_pow2(e1), up2 = kv4_pow2(e2);
#pragma unroll
                for (int i2 = 0; i2 < 8; i2++) x[i2] = x[i2] * up1 * up2;
                uint8_t *dst = smem + Cfg::Q + m * Cfg::TILE + (ch >> 3) * Cfg::HALF + r * 128 + (((ch & 7) ^ (r & 7)) << 4);
                *reinterpret_cast<uint4 *>(dst) = make_uint4(kv4_half2(x[0], x[4]), kv4_half2(x[1], x[5]),
                                                             kv4_half2(x[2], x[6]), kv4_half2(x[3], x[7]));
                if (ch == 0)  // never 0: masked scores are -inf times it
                    row_c[m * KP_M + r] = fmaxf(a.scale * 1.4426950408889634f * kv4_pow2(-e1) * kv4_pow2(-e2), FLT_MIN);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.q_full);

            const int r = (warp & 3) * 32 + lane, row = row0 + m * KP_M + r;
            const float cs = row_c[m * KP_M + r];
            const int t = a.pos0 + min(row, rows - 1) / G;  // the row's position
            const int t_lo = a.pos0 + (row0 + m * KP_M) / G, t_hi = a.pos0 + min(row0 + (m + 1) * KP_M - 1, rows - 1) / G;
            const int w_lo = a.window > 0 ? t - a.window : -1;  // positions above it are in the window
            const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
            const uint32_t ts = tmem + m * KP_N + lanes, to = tmem + 256 + m * HD + lanes;
            float ref = -INFINITY, l = 0.0f;
            for (int j = 0; j < n; j++) {
                KP_WAIT_WARP(bars.s_full[m], j & 1);
                tc::fence_after();
                const int p0 = seen.tile(tile0 + j) * KP_N;
                const bool whole = p0 + KP_N - 1 <= t_lo && (a.window == 0 || p0 > t_hi - a.window || p0 + KP_N <= a.n_sink);
                // P against `ref`, the largest score (scaled), the sum
                uint32_t p[KP_N / 2];
                auto attempt = [&](float neg_ref, float &mx, float &sum) {
                    mx = -INFINITY, sum = 0.0f;
                    float sum2 = 0.0f;
#pragma unroll
                    for (int ch = 0; ch < KP_N; ch += 32) {
                        uint32_t s[32];
                        tc::ld32(ts + ch, s);
                        tc::wait_ld();
                        if (!whole) {
#pragma unroll
                            for (int i = 0; i < 32; i++) {
                                const int k = p0 + ch + i;
                                if (k > t || (k <= w_lo && k >= a.n_sink)) s[i] = 0xff800000u;  // -inf
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            const float s0 = __uint_as_float(s[i]), s1 = __uint_as_float(s[i + 1]);
                            mx = fmaxf(mx, fmaxf(s0, s1));
                            const float e0 = kv4_exp2(fmaf(s0, cs, neg_ref)), e1 = kv4_exp2(fmaf(s1, cs, neg_ref));
                            sum += e0, sum2 += e1;
                            p[(ch + i) / 2] = kv4_half2(e0, e1);
                        }
                    }
                    mx *= cs;
                    sum += sum2;
                };
                float mx, sum;
                attempt(KP_BIAS - (ref == -INFINITY ? 0.0f : ref), mx, sum);
                if (__any_sync(0xffffffffu, mx > ref + KP_ROOM || (mx > -INFINITY && ref == -INFINITY))) {
                    const float next = fmaxf(ref, mx);
                    const float f = ref == -INFINITY ? 0.0f : kv4_exp2(ref - next);
                    ref = next;
                    l *= f;
                    if (j > 0) {
#pragma unroll 1
                        for (int ch = 0; ch < HD; ch += 32) {
                            uint32_t o[32];
                            tc::ld32(to + ch, o);
                            tc::wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                            tc::st32(to + ch, o);
                        }
                    }
                    attempt(KP_BIAS - (ref == -INFINITY ? 0.0f : ref), mx, sum);
                }
                l += sum;
                tc::st32(ts, p);
                tc::st32(ts + 32, p + 32);
                tc::wait_st();
                tc::fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars.p_full[m]);
            }
            // ---- the rows' results
            float inv = l == 0.0f ? 0.0f : 1.0f / l;
            float *part = nullptr;
            if (a.splits > 1) {
                part = a.part + ((int64_t)blockIdx.x * KP_ROWS + m * KP_M + r) * (HD + 2);
                part[0] = ref, part[1] = l;
                inv = 1.0f;
            }
            if (n > 0) {
                KP_WAIT_WARP(bars.o_full[m], 0);
                tc::fence_after();
                T *out = reinterpret_cast<T *>(a.out) + (int64_t)(row / G) * a.out_ld + (int64_t)(g * G + row % G) * HD;
#pragma unroll 1
                for (int ch = 0; ch < HD; ch += 32) {
                    uint32_t o[32];
                    tc::ld32(to + ch, o);
                    tc::wait_ld();
                    if (row < rows) {
#pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            // column 2e of a chunk is value e, column 2e + 1 value 4 + e
                            float x[8];
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                x[e] = __uint_as_float(o[i + 2 * e]) * inv, x[4 + e] = __uint_as_float(o[i + 2 * e + 1]) * inv;
                            if (part) {
#pragma unroll
                                for (int e = 0; e < 8; e += 2)
                                    *reinterpret_cast<float2 *>(part + 2 + ch + i + e) = make_float2(x[e], x[e + 1]);
                            } else {
                                kv4_store_row(out + ch + i, x);
                            }
                        }
                    }
                }
            }
        }
    } else if (warp < 12) {
        // ------------------------------------------------------------ dequantise: a thread per position
        const int r = threadIdx.x - 256;
        const __half2 cap = __float2half2_rn(KP_SCALE_MAX), ncap = __float2half2_rn(-KP_SCALE_MAX);
        for (int i = 0; i < 2 * n; i++) {
            const int j = i >> 1, slot = j & 1, rs = i % KP_RAW;
            const bool is_v = i & 1;
            uint8_t *dst = smem + (is_v ? Cfg::V : Cfg::K) + slot * Cfg::TILE;
            KP_WAIT_WARP(bars.raw_full[rs], (i / KP_RAW) & 1);
            if (j >= 2) KP_WAIT_WARP(is_v ? bars.v_empty[slot] : bars.k_empty[slot], ((j >> 1) - 1) & 1);
            const uint8_t *raw = smem + Cfg::R + rs * Cfg::RAW;
            const int pos = seen.tile(tile0 + j) * KP_N + r;
            uint32_t sc[NB / 2];
#pragma unroll
            for (int b = 0; b < NB / 2; b++) {
                sc[b] = *reinterpret_cast<const uint32_t *>(raw + Cfg::CODES + (r * NB + 2 * b) * 2);
                __half2 h;
                memcpy(&h, &sc[b], 4);
                h = __hmax2(__hmin2(h, cap), ncap);  // also keeps a NaN out
                memcpy(&sc[b], &h, 4);
                if (!seen.sees(pos, a.n_sink)) sc[b] = 0;  // a row that no query sees may hold anything
            }
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const uint4 w = *reinterpret_cast<const uint4 *>(raw + r * (HD / 2) + 16 * (b ^ kv4_turn<HD>(r)));
                __half2 d;
                const uint32_t dd = __byte_perm(sc[b / 2], 0, b & 1 ? 0x3232 : 0x1010);
                memcpy(&d, &dd, 4);
                uint8_t *half = dst + (b >> 1) * Cfg::HALF + r * 128;
                const int c0 = (b & 1) * 4;
                *reinterpret_cast<uint4 *>(half + (((c0 + 0) ^ (r & 7)) << 4)) = kp_word(w.x, d);
                *reinterpret_cast<uint4 *>(half + (((c0 + 1) ^ (r & 7)) << 4)) = kp_word(w.y, d);
                *reinterpret_cast<uint4 *>(half + (((c0 + 2) ^ (r & 7)) << 4)) = kp_word(w.z, d);
                *reinterpret_cast<uint4 *>(half + (((c0 + 3) ^ (r & 7)) << 4)) = kp_word(w.w, d);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&bars.raw_empty[rs]);
                mbar_arrive(is_v ? &bars.v_full[slot] : &bars.k_full[slot]);
            }
        }
    } else if (warp == 12) {
        // ------------------------------------------------------------ the MMAs
        if (lane == 0 && n > 0) {
            constexpr uint32_t id_qk = tc::idesc(KP_M, KP_N, false), id_pv = tc::idesc(KP_M, HD, true);
            const uint32_t q_at = smem_u32(smem + Cfg::Q), k_at = smem_u32(smem + Cfg::K), v_at = smem_u32(smem + Cfg::V);
            auto qk = [&](int m, int j) {
#pragma unroll
                for (int k = 0; k < HD / 16; k++) {
                    const uint32_t off = (k >> 2) * Cfg::HALF + (k & 3) * 32;
                    tc::mma_ss(tmem + m * KP_N, tc::desc_kmajor(q_at + m * Cfg::TILE + off),
                               tc::desc_kmajor(k_at + (j & 1) * Cfg::TILE + off), id_qk, k > 0);
                }
                tc::commit(&bars.s_full[m]);
            };
            auto pv = [&](int m, int j) {
#pragma unroll
                for (int k = 0; k < KP_N / 16; k++)
                    tc::mma_ts(tmem + 256 + m * HD, tmem + m * KP_N + 8 * k,
                               tc::desc_mnmajor(v_at + (j & 1) * Cfg::TILE + k * 2048, Cfg::HALF), id_pv, (j | k) > 0);
            };
            KP_WAIT(bars.q_full, 0);
            KP_WAIT(bars.k_full[0], 0);
            tc::fence_after();
            for (int m = 0; m < mt; m++) qk(m, 0);
            tc::commit(&bars.k_empty[0]);
            for (int j = 0; j < n; j++) {
                KP_WAIT(bars.v_full[j & 1], (j >> 1) & 1);
                for (int m = 0; m < mt; m++) {
                    KP_WAIT(bars.p_full[m], j & 1);
                    tc::fence_after();
                    pv(m, j);
                    if (m == mt - 1) tc::commit(&bars.v_empty[j & 1]);
                    if (j + 1 == n) {
                        tc::commit(&bars.o_full[m]);
                    } else {
                        if (m == 0) KP_WAIT(bars.k_full[(j + 1) & 1], ((j + 1) >> 1) & 1);
                        tc::fence_after();
                        qk(m, j + 1);
                        if (m == mt - 1) tc::commit(&bars.k_empty[(j + 1) & 1]);
                    }
                }
            }
        }
    } else {
        // ------------------------------------------------------------ raw tiles by bulk copies
        if (lane == 0) {
            const int64_t head = ((int64_t)a.seq * c.n_kv + g) * c.n_ctx;
            for (int i = 0; i < 2 * n; i++) {
                const int rs = i % KP_RAW;
                if (i >= KP_RAW) KP_WAIT(bars.raw_empty[rs], ((i / KP_RAW) - 1) & 1);
                const int p0 = seen.tile(tile0 + (i >> 1)) * KP_N;
                const int np = min(KP_N, c.n_ctx - p0);  // the cache may end inside the last tile (at 64)
                uint8_t *dst = smem + Cfg::R + rs * Cfg::RAW;
                mbar_arrive_expect_tx(&bars.raw_full[rs], (uint32_t)(np * (HD / 2 + NB * 2)));
                bulk_g2s(dst, (i & 1 ? c.vc : c.kc) + (head + p0) * (HD / 2), (uint32_t)(np * (HD / 2)), &bars.raw_full[rs]);
                bulk_g2s(dst + Cfg::CODES, (i & 1 ? c.vs : c.ks) + (head + p0) * NB, (uint32_t)(np * NB * 2),
                         &bars.raw_full[rs]);
            }
        }
    }
done:
    __syncwarp();
    tc::fence_before();
    __syncthreads();
    if (warp == 12) {
        tc::fence_after();
        tc::dealloc(tmem, 512);
    }
}

// The rows' parts, in order: a warp per row.
template <int HD, typename T>
__global__ void __launch_bounds__(256) kv4_join_kernel(const float *__restrict__ part, T *__restrict__ out, int64_t out_ld,
                                                       int n_tok, int n_head, int n_kv, int splits) {
    constexpr int V = HD / 32;  // values a lane
    pdl_wait();
    pdl_trigger();
    const int G = n_head / n_kv, rows = n_tok * G;
    const int64_t u = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (u >= (int64_t)rows * n_kv) return;
    const int g = (int)(u / rows), row = (int)(u % rows);
    const int blocks = (rows + KP_ROWS - 1) / KP_ROWS;
    const int64_t cta = ((int64_t)(blocks - 1 - row / KP_ROWS) * n_kv + g) * splits;
    const float *p = part + (cta * KP_ROWS + row % KP_ROWS) * (HD + 2);
    const int64_t step = (int64_t)KP_ROWS * (HD + 2);
    // lane s (and s + 32, ...) looks at part s
    float top = -INFINITY;
    for (int s = lane; s < splits; s += 32) top = fmaxf(top, __ldcg(p + s * step));
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float L = 0.0f, x[V];
#pragma unroll
    for (int i = 0; i < V; i++) x[i] = 0.0f;
#pragma unroll 4
    for (int s = 0; s < splits; s++) {
        const float2 rl = __ldcg(reinterpret_cast<const float2 *>(p + s * step));
        if (rl.y == 0.0f) continue;  // nothing seen there: its sums were not written
        const float f = rl.x == -INFINITY ? 1.0f : kv4_exp2(rl.x - top);
        L += f * rl.y;
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            const float2 y = __ldcg(reinterpret_cast<const float2 *>(p + s * step + 2 + V * lane + i));
            x[i] += f * y.x, x[i + 1] += f * y.y;
        }
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    T *o = out + (int64_t)(row / G) * out_ld + (int64_t)(g * G + row % G) * HD + V * lane;
#pragma unroll
    for (int i = 0; i < V; i += 2) {
        if constexpr (sizeof(T) == 4)
            *reinterpret_cast<float2 *>(o + i) = make_float2(x[i] * inv, x[i + 1] * inv);
        else
            *reinterpret_cast<uint32_t *>(o + i) = kv4_pack_bf2(x[i] * inv, x[i + 1] * inv);
    }
}

// ------------------------------------------------------------------ launchers
size_t kv4_prefill_part_bytes(int sm_count) { return (size_t)sm_count * KP_ROWS * (128 + 2) * 4; }

template <int HD, typename T>
static cudaError_t prefill_launch(const Kv4Attn &x, const Kv4Planes &c, float *part, int sm_count, int *err,
                                  cudaStream_t st) {
    using Cfg = Kv4PrefillCfg<HD>;
    static int set[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!set[dev]) {
        const cudaError_t e =
            cudaFuncSetAttribute(kv4_prefill_kernel<HD, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM);
        if (e != cudaSuccess) return e;
        set[dev] = 1;
    }
    const int G = x.n_head / c.n_kv;
    const int64_t rows = (int64_t)x.n_tok * G, blocks = (rows + KP_ROWS - 1) / KP_ROWS, ctas = blocks * c.n_kv;
    if (rows > (1 << 30)) return cudaErrorInvalidValue;
    // fewer CTAs than SMs: each block's positions over several, two tiles each at least
    const int tiles = kp_seen(x.pos0, 0, x.n_tok - 1, x.window, x.n_sink).tiles;
    int64_t splits = sm_count / ctas;
    if (splits > tiles / 2) splits = tiles / 2;
    if (splits < 1) splits = 1;
    Kv4PrefillArgs a;
    a.q = x.q, a.out = x.out, a.q_ld = x.q_ld, a.out_ld = x.out_ld;
    a.seq = x.seq0, a.pos0 = x.pos0, a.n_tok = x.n_tok, a.n_head = x.n_head;
    a.window = x.window, a.n_sink = x.n_sink, a.splits = (int)splits, a.scale = x.scale;
    a.part = part, a.err = err;
    cudaError_t e = launch_k(kv4_prefill_kernel<HD, T>, dim3((unsigned)(ctas * splits)), dim3(KP_THREADS),
                             (size_t)Cfg::SMEM, st, a, c);
    if (e != cudaSuccess || splits == 1) return e;
    return launch_k(kv4_join_kernel<HD, T>, dim3((unsigned)((rows * c.n_kv + 7) / 8)), dim3(256), 0, st,
                    (const float *)part, (T *)x.out, x.out_ld, x.n_tok, x.n_head, c.n_kv, (int)splits);
}

cudaError_t launch_kv4_prefill(bool f32, int head_dim, const Kv4Attn &x, const Kv4Planes &c, void *scratch,
                               int sm_count, int *err, cudaStream_t st) {
    if (x.n_tok <= 0) return cudaSuccess;
    float *part = kv4_scratch_parts(scratch, sm_count);
    if (head_dim == 128)
        return f32 ? prefill_launch<128, float>(x, c, part, sm_count, err, st)
                   : prefill_launch<128, __nv_bfloat16>(x, c, part, sm_count, err, st);
    return f32 ? prefill_launch<64, float>(x, c, part, sm_count, err, st)
               : prefill_launch<64, __nv_bfloat16>(x, c, part, sm_count, err, st);
}

}  // namespace tmoe
