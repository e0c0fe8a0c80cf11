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
// Warps: 0-3 and 4-7 the softmax of A and B, 8-11 dequantise K and 12-15 V, 16 issues the MMAs, 17 the
// bulk copies.  While the softmax of one tile runs, the tensor cores work on the other.
//
// Bound: per 256 rows x 128 positions of 128-wide heads the MMAs take 2048 clocks and so do the exps (16 a
// clock and SM); the dequantisation (13 instructions for 8 values, about 475 issue slots a scheduler)
// hides beside them.
//   - A code under a mask is 1024 + c in f16; minus 1032, times the block's scale: f16(d (c - 8)).  The pairs that
//     fall out of a word are values (0, 4), (1, 5), (2, 6), (3, 7); Q's chunks are written in that order,
//     and O's columns come out in it.
//   - The running reference of a row moves only when P against it adds up to more than 2^14 in half a tile (P is 2^6
//     at the reference, so that no P leaves f16 before that): no maximum is taken, and O needs no rescaling.
//     A tile is first tried with the old reference, S still whole in TMEM; the rare failure is redone.
//   - Q is scaled per row by a power of two into f16's range.  Scales are held to what f16 can carry times 8.
//   - Few query rows leave SMs idle, so their positions are split over CTAs, and kv4_join_kernel adds the parts.
#include "kernels.cuh"
#include "kv4.cuh"
#include "tcgen05.cuh"

namespace tmoe {

constexpr int KP_M = 128;            // rows of a tile
constexpr int KP_ROWS = 2 * KP_M;    // of a CTA
constexpr int KP_N = 128;            // positions of a tile
constexpr int KP_THREADS = 640;
// Registers per thread: the softmax warps take what the others give back (5 * 96 at launch)
constexpr int KP_REGS_SOFTMAX = 152, KP_REGS_DEQUANT = 64, KP_REGS_ISSUE = 48;
static_assert(2 * KP_REGS_SOFTMAX + 2 * KP_REGS_DEQUANT + KP_REGS_ISSUE <= 5 * 96, "the block's registers");
constexpr int KP_RAW = 3;            // raw tiles (of K or of V) in flight
constexpr float KP_BIAS = 6.0f;      // P is 2^KP_BIAS at the reference
constexpr float KP_MOST = 16384.0f;  // a half tile's sum of P above which the row's reference moves
constexpr float KP_SCALE_MAX = 8188.0f;  // 8 * this is f16's largest

struct Kv4PrefillArgs {
    const void *q;
    void *out;
    int64_t q_ld, out_ld;
    int seq, pos0, n_tok, n_head, window, n_sink, splits;
    float scale;
    float *part;  // splits > 1: [cta] of O as [HD / 4][KP_ROWS][4], then the references and sums as [2][KP_ROWS]
    int *err;
};

template <int HD>
struct Kv4PrefillCfg {
    static constexpr int NB = HD / 32, HALVES = HD / 64;  // 64-wide halves of a row: 128 bytes of f16
    static constexpr int HALF = KP_N * 128;               // bytes of a half tile
    static constexpr int TILE = HALVES * HALF;
    static constexpr int CODES = KP_N * HD / 2, SCALES = KP_N * NB * 2, RAW = CODES + SCALES;
    static constexpr int Q = 0, K = 2 * TILE, V = K + 2 * TILE, R = V + 2 * TILE, BARS = R + KP_RAW * RAW;
    static constexpr int SMEM = BARS + 256 + 1024 /* alignment */;
};

struct KpBars {
    uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], raw_empty[KP_RAW], s_full[2],
        p_full[2][2], o_half[2], o_full[2];
    // a slot holds K and V by turns; each of the two has its own barrier of it, so that its readers see every phase
    uint64_t raw_full[2][KP_RAW];
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

// 2^x of a pair
__device__ __forceinline__ float2 kp_exp2_pair(uint64_t x) {
    const float2 f = tc::unpair(x);
    return make_float2(kv4_exp2(f.x), kv4_exp2(f.y));
}

struct KpYes {
    static constexpr bool value = true;
};
struct KpNo {
    static constexpr bool value = false;
};

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
            mbar_init(&bars.p_full[i][0], 4);
            mbar_init(&bars.p_full[i][1], 4);
            mbar_init(&bars.o_half[i], 1);
            mbar_init(&bars.o_full[i], 1);
        }
        for (int i = 0; i < KP_RAW; i++) {
            mbar_init(&bars.raw_full[0][i], 1);
            mbar_init(&bars.raw_full[1][i], 1);
            mbar_init(&bars.raw_empty[i], 4);
        }
        fence_barrier_init();
    }
    if (warp == 16) tc::alloc(&bars.tmem, 512);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = bars.tmem;
    pdl_wait();
    pdl_trigger();

    if (warp < 8) {
        tc::more_registers<KP_REGS_SOFTMAX>();
        // ------------------------------------------------------------ Q, then the softmax: a thread per row
        const int m = warp >> 2;
        if (m < mt) {
            // The warp's 32 rows into the operand's layout, a thread per row: bf16 by asynchronous copies, all in flight,
            // and then in place; f32 read twice.  Loops stay rolled: their code is fetched anew by every CTA.
            uint8_t *q_tile = smem + Cfg::Q + m * Cfg::TILE;
            auto chunk = [&](int r, int ch) { return q_tile + (ch >> 3) * Cfg::HALF + r * 128 + (((ch & 7) ^ (r & 7)) << 4); };
            const int my_r = (warp & 3) * 32 + lane, my_row = min(row0 + m * KP_M + my_r, rows - 1);
            const T *my_q = reinterpret_cast<const T *>(a.q) + (int64_t)(my_row / G) * a.q_ld + (int64_t)(g * G + my_row % G) * HD;
            constexpr int CH = HD / 8;
            float top = 0.0f;
            if constexpr (sizeof(T) == 2) {
#pragma unroll 4
                for (int i = 0; i < 32; i += 32 / CH) {
                    const int src = i + lane / CH, ch = lane % CH;
                    const T *p = reinterpret_cast<const T *>(__shfl_sync(0xffffffffu, (unsigned long long)my_q, src)) + 8 * ch;
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(chunk((warp & 3) * 32 + src, ch))), "l"(p)
                                 : "memory");
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
                asm volatile("cp.async.wait_group 0;" ::: "memory");
                __syncwarp();
#pragma unroll 2
                for (int ch = 0; ch < CH; ch++) {
                    const uint4 u = *reinterpret_cast<const uint4 *>(chunk(my_r, ch));
                    // magnitudes of bf16 order as their bits
                    const uint32_t h = __vmaxu2(__vmaxu2(u.x & 0x7fff7fffu, u.y & 0x7fff7fffu),
                                                __vmaxu2(u.z & 0x7fff7fffu, u.w & 0x7fff7fffu));
                    top = fmaxf(top, fmaxf(__uint_as_float(h << 16), __uint_as_float(h & 0xffff0000u)));
                }
            } else {
#pragma unroll 2
                for (int ch = 0; ch < CH; ch++) {
                    float x[8];
                    kv4_load_row(my_q + 8 * ch, x);
#pragma unroll
                    for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[e]));
                }
            }
            // 2^e * top in [2^5, 2^6): exact for bf16 values down to 2^-22 of the largest
            const int e = top > 0.0f && top <= FLT_MAX ? 5 - ilogbf(top) : 0;
            const int e1 = e / 2, e2 = e - e1;
            const float up1 = kv4_pow2(e1), up2 = kv4_pow2(e2);
#pragma unroll 2
            for (int ch = 0; ch < CH; ch++) {
                uint4 *dst = reinterpret_cast<uint4 *>(chunk(my_r, ch));
                float x[8];
                if constexpr (sizeof(T) == 2) {
                    const uint4 u = *dst;
                    kv4_bf2(u.x, x[0], x[1]), kv4_bf2(u.y, x[2], x[3]), kv4_bf2(u.z, x[4], x[5]), kv4_bf2(u.w, x[6], x[7]);
                } else {
                    kv4_load_row(my_q + 8 * ch, x);
                }
#pragma unroll
                for (int v = 0; v < 8; v++) x[v] = x[v] * up1 * up2;
                *dst = make_uint4(kv4_half2(x[0], x[4]), kv4_half2(x[1], x[5]), kv4_half2(x[2], x[6]), kv4_half2(x[3], x[7]));
            }
            // log2 score of an accumulator's 1; never 0: masked scores are -inf times it
            const float cs = fmaxf(a.scale * 1.4426950408889634f * kv4_pow2(-e1) * kv4_pow2(-e2), FLT_MIN);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.q_full);

            const int r = my_r, row = row0 + m * KP_M + r;
            const int t = a.pos0 + min(row, rows - 1) / G;  // the row's position
            const int t_lo = a.pos0 + (row0 + m * KP_M) / G, t_hi = a.pos0 + min(row0 + (m + 1) * KP_M - 1, rows - 1) / G;
            const int w_lo = a.window > 0 ? t - a.window : -1;  // positions above it are in the window
            const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
            const uint32_t ts = tmem + m * KP_N + lanes, to = tmem + 256 + m * HD + lanes;
            float ref = -INFINITY, l = 0.0f;
            // P of 32 columns of S against a reference (exponents s c + r), and its sum; positions from k0 on
            auto exps = [&](const uint32_t (&s)[32], uint32_t *p, uint64_t c2, uint64_t r2, uint64_t (&sum)[2], int k0, auto masked) {
                // by stages over all 32: a group at a time would wait for each result
                uint64_t x[16];
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    uint32_t v[2] = {s[2 * i], s[2 * i + 1]};
                    if constexpr (decltype(masked)::value) {
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            const int k = k0 + 2 * i + u;
                            if (k > t || (k <= w_lo && k >= a.n_sink)) v[u] = 0xff800000u;  // -inf
                        }
                    }
                    x[i] = tc::fma2(tc::pair(__uint_as_float(v[0]), __uint_as_float(v[1])), c2, r2);
                }
                float2 e[16];
#pragma unroll
                for (int i = 0; i < 16; i++) e[i] = kp_exp2_pair(x[i]);
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    sum[i & 1] = tc::add2(sum[i & 1], tc::pair(e[i].x, e[i].y));
                    p[i] = kv4_half2(e[i].x, e[i].y);
                }
            };
            uint32_t s0[32], s1[32], p[32];  // 64 columns of S, and their P
#pragma unroll 1
            for (int j = 0; j < n; j++) {
                KP_WAIT_WARP(bars.s_full[m], j & 1);
                tc::fence_after();
                tc::ld32(ts, s0);
                // In halves of 64 positions, so that the first one's product runs beside the second's exps; half of the
                // next 64 columns is read while the second half of these is worked on
#pragma unroll 1
                for (int hf = 0; hf < 2; hf++) {
                    const int k0 = seen.tile(tile0 + j) * KP_N + 64 * hf;
                    const bool whole = k0 + 63 <= t_lo && (a.window == 0 || k0 > t_hi - a.window || k0 + 64 <= a.n_sink);
                    const uint32_t th = ts + 64 * hf;
                    tc::ld32(th + 32, s1);
                    tc::wait_ld(s0);
                    tc::wait_ld(s1);
                    float sum;
                    bool raise = __any_sync(0xffffffffu, ref == -INFINITY);
#pragma unroll 1
                    for (int tries = 0; tries < 2; tries++) {
                        if (raise) {
                            tries = 1;
                            float mx = -INFINITY;
#pragma unroll 1
                            for (int ch = 0; ch < 64; ch += 32) {
                                tc::ld32(th + ch, s0);
                                tc::wait_ld(s0);
#pragma unroll
                                for (int i = 0; i < 32; i++) {
                                    const int k = k0 + ch + i;
                                    if (k <= t && (k > w_lo || k < a.n_sink)) mx = fmaxf(mx, __uint_as_float(s0[i]));
                                }
                            }
                            const float next = fmaxf(ref, mx * cs);
                            const float f = ref == -INFINITY ? 0.0f : kv4_exp2(ref - next);
                            ref = next;
                            l *= f;
                            if (hf) {  // the first half's product has to be in O
                                KP_WAIT_WARP(bars.o_half[m], j & 1);
                                tc::fence_after();
                            }
                            if (j > 0 || hf) {
#pragma unroll 1
                                for (int ch = 0; ch < HD; ch += 32) {
                                    tc::ld32(to + ch, s0);
                                    tc::wait_ld(s0);
#pragma unroll
                                    for (int i = 0; i < 32; i++) s0[i] = __float_as_uint(__uint_as_float(s0[i]) * f);
                                    tc::st32(to + ch, s0);
                                }
                            }
                            tc::ld32(th, s0);
                            tc::ld32(th + 32, s1);
                            tc::wait_ld(s0);
                            tc::wait_ld(s1);
                        }
                        const float neg_ref = KP_BIAS - (ref == -INFINITY ? 0.0f : ref);
                        const uint64_t c2 = tc::pair(cs, cs), r2 = tc::pair(neg_ref, neg_ref);
                        uint64_t sums[2] = {0, 0};
                        if (whole)
                            exps(s0, p, c2, r2, sums, k0, KpNo{});
                        else
                            exps(s0, p, c2, r2, sums, k0, KpYes{});
                        if (!hf) tc::ld32(ts + 64, s0);
                        if (whole)
                            exps(s1, p + 16, c2, r2, sums, k0 + 32, KpNo{});
                        else
                            exps(s1, p + 16, c2, r2, sums, k0 + 32, KpYes{});
                        const float2 x = tc::unpair(tc::add2(sums[0], sums[1]));
                        sum = x.x + x.y;
                        raise = __any_sync(0xffffffffu, sum > KP_MOST);
                        if (!raise) break;
                        tc::wait_ld(s0);
                    }
                    l += sum;
                    tc::st32(th, p);
                    tc::wait_st();
                    tc::fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bars.p_full[m][hf]);
                }
            }
            // ---- the rows' results
            float inv = l == 0.0f ? 0.0f : 1.0f / l;
            float *part = nullptr;
            if (a.splits > 1) {  // O as it is, rows side by side
                part = a.part + (int64_t)blockIdx.x * KP_ROWS * (HD + 2) + (m * KP_M + r) * 4;
                float *stats = a.part + (int64_t)blockIdx.x * KP_ROWS * (HD + 2) + KP_ROWS * HD + m * KP_M + r;
                stats[0] = ref, stats[KP_ROWS] = l;
            }
            if (n > 0) {
                KP_WAIT_WARP(bars.o_full[m], 0);
                tc::fence_after();
                T *out = reinterpret_cast<T *>(a.out) + (int64_t)(row / G) * a.out_ld + (int64_t)(g * G + row % G) * HD;
#pragma unroll 1
                for (int ch = 0; ch < HD; ch += 32) {
                    uint32_t o[32];
                    tc::ld32(to + ch, o);
                    tc::wait_ld(o);
                    if (part) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            *reinterpret_cast<uint4 *>(part + (ch + i) * KP_ROWS) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                    } else if (row < rows) {
#pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            // column 2e of a chunk is value e, column 2e + 1 value 4 + e
                            float x[8];
#pragma unroll
                            for (int v = 0; v < 4; v++)
                                x[v] = __uint_as_float(o[i + 2 * v]) * inv, x[4 + v] = __uint_as_float(o[i + 2 * v + 1]) * inv;
                            kv4_store_row(out + ch + i, x);
                        }
                    }
                }
            }
        }
    } else if (warp < 16) {
        tc::fewer_registers<KP_REGS_DEQUANT>();
        // ------------------------------------------------------------ dequantise: a thread per position
        const int r = threadIdx.x & 127;
        const bool is_v = warp >= 12;
        const __half2 cap = __float2half2_rn(KP_SCALE_MAX), ncap = __float2half2_rn(-KP_SCALE_MAX);
        for (int j = 0; j < n; j++) {
            const int i = 2 * j + is_v, slot = j & 1, rs = i % KP_RAW;
            uint8_t *dst = smem + (is_v ? Cfg::V : Cfg::K) + slot * Cfg::TILE;
            KP_WAIT_WARP(bars.raw_full[is_v][rs], (j / KP_RAW) & 1);
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
    } else {
        tc::fewer_registers<KP_REGS_ISSUE>();
        if (warp == 16) {
            // -------------------------------------------------------- the MMAs
            if (n > 0) {
                constexpr uint32_t id_qk = tc::idesc(KP_M, KP_N, false), id_pv = tc::idesc(KP_M, HD, true);
                const uint32_t q_lo = tc::desc_lo(smem_u32(smem + Cfg::Q), 16), k_lo = tc::desc_lo(smem_u32(smem + Cfg::K), 16),
                               v_lo = tc::desc_lo(smem_u32(smem + Cfg::V), Cfg::HALF);
                auto qk = [&](int m, int j) {
                    const uint32_t a_lo = q_lo + m * (Cfg::TILE >> 4), b_lo = k_lo + (j & 1) * (Cfg::TILE >> 4);
                    if (tc::elect()) {
#pragma unroll
                        for (int k = 0; k < HD / 16; k++) {
                            const uint32_t off = ((k >> 2) * Cfg::HALF + (k & 3) * 32) >> 4;
                            tc::mma_ss(tmem + m * KP_N, a_lo + off, tc::DESC_HI, b_lo + off, tc::DESC_HI, id_qk, k > 0);
                        }
                        tc::commit(&bars.s_full[m]);
                    }
                    __syncwarp();
                };
                auto pv = [&](int m, int j, int hf) {
                    const uint32_t b_lo = v_lo + (j & 1) * (Cfg::TILE >> 4) + hf * (64 * 128 >> 4);
                    if (tc::elect()) {
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            tc::mma_ts(tmem + 256 + m * HD, tmem + m * KP_N + 64 * hf + 8 * k, b_lo + k * (2048 >> 4), tc::DESC_HI,
                                       id_pv, k > 0 ? 1 : j | hf);
                        if (hf == 0) {
                            tc::commit(&bars.o_half[m]);
                        } else {
                            if (m == mt - 1) tc::commit(&bars.v_empty[j & 1]);
                            if (j + 1 == n) tc::commit(&bars.o_full[m]);
                        }
                    }
                    __syncwarp();
                };
                KP_WAIT_WARP(bars.q_full, 0);
                KP_WAIT_WARP(bars.k_full[0], 0);
                tc::fence_after();
                for (int m = 0; m < mt; m++) qk(m, 0);
                if (tc::elect()) tc::commit(&bars.k_empty[0]);
                for (int j = 0; j < n; j++) {
                    KP_WAIT_WARP(bars.v_full[j & 1], (j >> 1) & 1);
                    for (int m = 0; m < mt; m++) {
                        for (int hf = 0; hf < 2; hf++) {
                            KP_WAIT_WARP(bars.p_full[m][hf], j & 1);
                            tc::fence_after();
                            pv(m, j, hf);
                        }
                        if (j + 1 < n) {
                            if (m == 0) KP_WAIT_WARP(bars.k_full[(j + 1) & 1], ((j + 1) >> 1) & 1);
                            tc::fence_after();
                            qk(m, j + 1);
                            if (m == mt - 1 && tc::elect()) tc::commit(&bars.k_empty[(j + 1) & 1]);
                        }
                    }
                }
            }
        } else if (warp == 17) {
        // ------------------------------------------------------------ raw tiles by bulk copies
        if (lane == 0) {
            const int64_t head = ((int64_t)a.seq * c.n_kv + g) * c.n_ctx;
            for (int i = 0; i < 2 * n; i++) {
                const int rs = i % KP_RAW;
                if (i >= KP_RAW) KP_WAIT(bars.raw_empty[rs], ((i / KP_RAW) - 1) & 1);
                const int p0 = seen.tile(tile0 + (i >> 1)) * KP_N;
                const int np = min(KP_N, c.n_ctx - p0);  // the cache may end inside the last tile (at 64)
                uint8_t *dst = smem + Cfg::R + rs * Cfg::RAW;
                uint64_t *full = &bars.raw_full[i & 1][rs];
                mbar_arrive_expect_tx(full, (uint32_t)(np * (HD / 2 + NB * 2)));
                bulk_g2s(dst, (i & 1 ? c.vc : c.kc) + (head + p0) * (HD / 2), (uint32_t)(np * (HD / 2)), full);
                bulk_g2s(dst + Cfg::CODES, (i & 1 ? c.vs : c.ks) + (head + p0) * NB, (uint32_t)(np * NB * 2),
                         full);
            }
        }
        }
    }
done:
    __syncwarp();
    tc::fence_before();
    __syncthreads();
    if (warp == 16) {
        tc::fence_after();
        tc::dealloc(tmem, 512);
    }
}

// The rows' parts, in order: a thread per row and 8 values, a block's rows side by side.
template <int HD, typename T>
__global__ void __launch_bounds__(KP_ROWS) kv4_join_kernel(const float *__restrict__ part, T *__restrict__ out, int64_t out_ld,
                                                           int n_tok, int n_head, int n_kv, int splits) {
    pdl_wait();
    pdl_trigger();
    const int G = n_head / n_kv, rows = n_tok * G, blocks = (rows + KP_ROWS - 1) / KP_ROWS;
    const int g8 = blockIdx.x % (HD / 8), list = blockIdx.x / (HD / 8);  // of (block, KV head), as the CTAs were numbered
    const int row = (blocks - 1 - list / n_kv) * KP_ROWS + (int)threadIdx.x, g = list % n_kv;
    if (row >= rows) return;
    constexpr int64_t STEP = (int64_t)KP_ROWS * (HD + 2);
    const float *p = part + (int64_t)list * splits * STEP;
    const float *stats = p + KP_ROWS * HD + threadIdx.x;
    const float4 *o = reinterpret_cast<const float4 *>(p) + 2 * g8 * KP_ROWS + threadIdx.x;
    float top = -INFINITY, L = 0.0f, x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 1
    for (int s0 = 0; s0 < splits; s0 += 4) {
        float r[4], l[4];
        float4 y[4][2];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const bool in = s0 + u < splits;
            const int64_t at = (s0 + u) * STEP;
            r[u] = in ? __ldcg(stats + at) : -INFINITY, l[u] = in ? __ldcg(stats + at + KP_ROWS) : 0.0f;
            y[u][0] = in ? __ldcg(o + at / 4) : make_float4(0, 0, 0, 0);
            y[u][1] = in ? __ldcg(o + at / 4 + KP_ROWS) : make_float4(0, 0, 0, 0);
        }
        const float next = fmaxf(fmaxf(top, fmaxf(r[0], r[1])), fmaxf(r[2], r[3]));
        const float f = top == -INFINITY ? 1.0f : kv4_exp2(top - next);
        top = next, L *= f;
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] *= f;
#pragma unroll
        for (int u = 0; u < 4; u++) {
            if (l[u] == 0.0f) continue;  // nothing seen there: its sums were not written
            const float w = r[u] == -INFINITY ? 1.0f : kv4_exp2(r[u] - top);
            L += w * l[u];
            // column 2e of a chunk is value e, column 2e + 1 value 4 + e
            x[0] += w * y[u][0].x, x[4] += w * y[u][0].y, x[1] += w * y[u][0].z, x[5] += w * y[u][0].w;
            x[2] += w * y[u][1].x, x[6] += w * y[u][1].y, x[3] += w * y[u][1].z, x[7] += w * y[u][1].w;
        }
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] *= inv;
    kv4_store_row(out + (int64_t)(row / G) * out_ld + (int64_t)(g * G + row % G) * HD + 8 * g8, x);
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
    return launch_k(kv4_join_kernel<HD, T>, dim3((unsigned)(ctas * (HD / 8))), dim3(KP_ROWS), 0, st,
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
