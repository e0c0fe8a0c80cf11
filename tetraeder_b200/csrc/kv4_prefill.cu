// Attention of many query tokens of one sequence over the 4-bit KV cache (format: kv4.cuh), on the
// 5th-generation tensor cores.
//
// The query rows of a KV head are its tokens times the query heads that share it (row r: token r / G, head
// r % G), so that one dequantised tile of K and V serves all of them.  A block is 256 rows, as two
// 128-row tiles A and B; a CTA, one per SM, takes its share of the blocks (see KpItem) and walks the 128-position tiles that
// a block's tokens see:
//   S = Q K^T   tcgen05, Q and K f16 in shared memory (128-byte swizzle), S f32 in TMEM (128 columns a tile)
//   P           a thread per row: exp2(S c - ref) as f16, back into TMEM over S
//   O += P V    tcgen05, P from TMEM, V f16 in shared memory as it lies (rows are positions: an N-major
//               operand), O f32 in TMEM
// Warps: 0-3 and 4-7 the softmax of A and B, 8-11 dequantise K and load Q of A, 12-15 V and Q of B, 16 issues the MMAs, 17
// the bulk copies.  While the softmax of one tile runs, the tensor cores work on the other; the roles run on from one block into
// the next, so that a block's Q, first tiles and first S are ready when the last one's O is written.
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
//   - Q is scaled per row by a power of two into f16's range.
//   - A scale of 2^13 and more takes its values (up to 8 times f16's largest) out of f16.  The first pass over a CTA's run only notes
//     that it met one; the CTA then does its run again with K and V over 8.  Without one this costs a test of bits per scale.
//   - What a warp has alike (its role, its block, the conditions of a tile) goes through a shuffle from lane 0, and
//     shared memory is declared aligned: branches, addresses and descriptors then stay out of the lanes' registers (a tile
//     pair 2.41 us, without either 2.79).
//   - With f32 rows (f16_products) the operands are the same f16: 11 bits of Q, K, P and V, 4e-4 of the largest output off, where a
//     4-bit value is itself off by 1/16 of its block's largest.  Callers who want f32's precision get the decode kernel.
// Measured (32 heads over 4, width 128, bf16; graph replay): 8192 tokens 600 to 620 us by device, 890 to 915 TFLOP/s; 4097 tokens
// of 40 heads over 8 under a window of 4096 430 us; 2048 tokens 50 us (64-wide heads 43, f32 rows 69); 33 tokens at position
// 20000 36 us.  A tile pair takes about 4400 clocks, the softmax's chain of
// S wait (1000), TMEM loads, exps and P (1700 a half) for A beside the same for B; at length the device is at its power limit
// (1000 W, 1.83 GHz).
#include "kernels.cuh"
#include "kv4.cuh"
#include "tcgen05.cuh"

namespace tmoe {

constexpr int KP_M = 128;            // rows of a tile
constexpr int KP_ROWS = 2 * KP_M;    // of a block
constexpr int KP_N = 128;            // positions of a tile
constexpr int KP_THREADS = 640;
// Registers per thread: the softmax warps take what the others give back (5 * 96 at launch)
constexpr int KP_REGS_SOFTMAX = 144, KP_REGS_DEQUANT = 64, KP_REGS_ISSUE = 64;
static_assert(2 * KP_REGS_SOFTMAX + 2 * KP_REGS_DEQUANT + KP_REGS_ISSUE <= 5 * 96, "the block's registers");
constexpr int KP_RAW = 3;            // raw tiles (of K or of V) in flight
// Work (see KpItem) of a tile of positions, of one of a block without rows in B (33 tokens at 20000: 5 40 us, 6 36, 7 37), of a block
// itself (8192 tokens: 8 615 us, 12 597, 20 604), and how much longer a CTA may work to spare cuts and their join (1024
// tokens: 28 41 us, cut, 76 27, whole; 2048 tokens at 4096 differ by 92: cut 177 us, whole 194).
constexpr int KP_UNITS = 8, KP_UNITS1 = 6, KP_UNITS_BLOCK = 12, KP_UNITS_JOIN = 76;
constexpr int KP_MAX_CTAS = 512;
constexpr float KP_BIAS = 6.0f;      // P is 2^KP_BIAS at the reference
constexpr float KP_MOST = 16384.0f;  // a half tile's sum of P above which the row's reference moves
constexpr float KP_BIG = 8.0f, KP_BIG_LOG2 = 3.0f;  // K and V are held over this where they leave f16 (see KpBars::big)

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

// A block that was cut, and the first and last of the runs that share it
struct KpCut {
    int blk, g, first, last;  // first < 0: none
};
struct Kv4PrefillArgs {
    const void *q;
    void *out;
    int64_t q_ld, out_ld;
    int seq, pos0, n_tok, window, n_sink;
    int group, blocks, n_kv;  // query heads of a KV head; blocks of KP_ROWS rows of one
    bool whole;               // see KpItem
    uint64_t group_inv;       // floor((2^64 - 1) / group) + 1, or 0 for a group of 1
    int64_t head_units;       // a KV head's work (see KpItem)
    float scale;
    KpCut *cuts;  // of the second run of each block that was cut: [run - 1], or (by_item) [g * blocks + blk]
    bool by_item;
    float *part;  // [cta][head, tail of its run] of O as [HD / 4][KP_ROWS][4], then the references and sums as [2][KP_ROWS]
    int *err;
    // row / group, exact for rows below 2^32
    __device__ __forceinline__ int token(int row) const { return group_inv ? (int)__umul64hi((uint64_t)row, group_inv) : row; }
};

// A value that all lanes have alike
__device__ __forceinline__ int kp_uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

// The work is one list: KV head by KV head, block by block, tile by tile.  A block costs KP_UNITS_BLOCK, then a tile
// KP_UNITS (KP_UNITS1 where there are no rows in B).  Every CTA takes an even run of the list, so a block may be cut: its pieces
// go to `part` and kv4_join_kernel adds them.  Where whole blocks share out as well (see prefill_launch) nothing is cut: the CTAs
// take them in turn, the last (longest) ones first, to and fro.
struct KpItem {
    int g, blk, s;  // s: the block's first unit, from the run's first (whole: the turn)
    int row0, n_rows, tiles, tile0, n;
    Kv4Seen seen;
    __device__ __forceinline__ int mt() const { return n_rows > KP_M ? 2 : 1; }
    __device__ __forceinline__ bool uncut() const { return n == tiles; }
    __device__ __forceinline__ int tiles_before(int units) const {  // tiles that begin before the block's first `units`
        const int u = units - KP_UNITS_BLOCK;
        return u <= 0 ? 0 : min(tiles, mt() == 2 ? (u + KP_UNITS - 1) / KP_UNITS : (u + KP_UNITS1 - 1) / KP_UNITS1);
    }
    __device__ __forceinline__ int units() const { return KP_UNITS_BLOCK + tiles * (mt() == 2 ? KP_UNITS : KP_UNITS1); }
    // The part of this block in a run of `len` units: tiles tile0 .. tile0 + n - 1 of `tiles`; false: beyond the run
    __device__ __forceinline__ bool in_run(const Kv4PrefillArgs &a, int len) {
        if (a.whole) {
            const int ctas = (int)gridDim.x, i = s * ctas + (s & 1 ? ctas - 1 - (int)blockIdx.x : (int)blockIdx.x);
            if (i >= a.blocks * a.n_kv) return false;
            blk = a.blocks - 1 - i / a.n_kv, g = i % a.n_kv;
        } else if (s >= len) {
            return false;
        }
        row0 = blk * KP_ROWS, n_rows = min(KP_ROWS, a.n_tok * a.group - row0);
        seen = kp_seen(a.pos0, a.token(row0), a.token(row0 + n_rows - 1), a.window, a.n_sink);
        tiles = seen.tiles;
        tile0 = 0, n = tiles;
        if (!a.whole) tile0 = tiles_before(-s), n = tiles_before(len - s) - tile0;
        return true;
    }
    // The same by a whole warp, the results in uniform registers: what depends on them (branches, descriptors) is the
    // warp's then, not each lane's, and costs less
    __device__ __forceinline__ bool in_run_warp(const Kv4PrefillArgs &a, int len) {
        if (!__any_sync(0xffffffffu, in_run(a, len))) return false;
        for (int *x : {&g, &blk, &s, &row0, &n_rows, &tiles, &tile0, &n, &seen.len, &seen.from, &seen.head, &seen.body})
            *x = kp_uniform(*x);
        return true;
    }
    __device__ __forceinline__ void next(const Kv4PrefillArgs &a) {
        if (a.whole) {
            s++;
            return;
        }
        s += units();
        if (++blk == a.blocks) blk = 0, g++;
    }
};
// The run that holds a unit, of `ctas` runs that begin at total * cta / ctas
__device__ __forceinline__ int kp_run_of(int64_t unit, int64_t total, int ctas) {
    return (int)(((unit + 1) * ctas - 1) / total);
}

template <int HD>
struct Kv4PrefillCfg {
    static constexpr int NB = HD / 32, HALVES = HD / 64;  // 64-wide halves of a row: 128 bytes of f16
    static constexpr int HALF = KP_N * 128;               // bytes of a half tile
    static constexpr int TILE = HALVES * HALF;
    static constexpr int CODES = KP_N * HD / 2, SCALES = KP_N * NB * 2, RAW = CODES + SCALES;
    static constexpr int Q = 0, K = 2 * TILE, V = K + 2 * TILE, R = V + 2 * TILE, CS = R + KP_RAW * RAW, UP = CS + KP_ROWS * 4,
                         BARS = UP + KP_ROWS * 4;
    static constexpr int SMEM = BARS + 1024;
    static constexpr int64_t PART = KP_ROWS * (HD + 2);  // floats of a piece
};

struct KpBars {
    uint64_t q_full[2], q_empty[2], k_full[2], k_empty[2], v_full[2], v_empty[2], raw_empty[KP_RAW], s_full[2],
        p_full[2][2], o_half[2], o_full[2];
    // a slot holds K and V by turns; each of the two has its own barrier of it, so that its readers see every phase
    uint64_t raw_full[2][KP_RAW];
    uint32_t tmem;
    // A scale of 2^13 and more, 8 of which leave f16, was met: the CTA does its run a second time, K and V over KP_BIG
    int big;
    int failed;  // a wait ran out
    int g, blk, s, len;  // the run: its first block, that one's first unit from the run's first, its units
    KpCut cut;
    KpItem item[8];  // the softmax warps'
};
static_assert(sizeof(KpBars) <= 1024, "barrier room");

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

// The roles meet at the end of the first pass over the run (barrier 1)
__device__ __forceinline__ void kp_meet(bool wait) {
    if (wait)
        asm volatile("barrier.cta.sync 1, %0;" ::"n"(KP_THREADS) : "memory");
    else
        asm volatile("barrier.cta.arrive 1, %0;" ::"n"(KP_THREADS) : "memory");
}
// Bounded waits by a whole warp.  One that runs out latches the error and ends the role.
#define KP_WAIT_WARP(bar, phase)                                                            \
    do {                                                                                    \
        if (!__all_sync(0xffffffffu, mbar_wait_bounded(&(bar), (uint32_t)(phase)))) {       \
            if (lane == 0) latch_error(a.err, TMOE_DEV_ERR_TIMEOUT), bars.failed = 1;       \
            __syncwarp();                                                                   \
            if (!second) kp_meet(false);                                                    \
            goto done;                                                                      \
        }                                                                                   \
    } while (0)
template <int HD, typename T>
__global__ void __launch_bounds__(KP_THREADS, 1) kv4_prefill_kernel(const Kv4PrefillArgs a, const Kv4Planes c) {
    using Cfg = Kv4PrefillCfg<HD>;
    constexpr int NB = Cfg::NB;
    extern __shared__ __align__(1024) uint8_t smem[];  // as declared, so that addresses in it are constants
    if (smem_u32(smem) & 1023) {  // the swizzle needs it
        if (threadIdx.x == 0) latch_error(a.err, TMOE_DEV_ERR_TIMEOUT);
        return;
    }
    KpBars &bars = *reinterpret_cast<KpBars *>(smem + Cfg::BARS);
    const int warp = kp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        bars.big = bars.failed = 0;
        for (int i = 0; i < 2; i++) {
            mbar_init(&bars.q_full[i], 4);
            mbar_init(&bars.q_empty[i], 1 + 4);
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
    if (a.whole) {
        if (threadIdx.x == 0) bars.g = bars.blk = bars.s = bars.len = 0;
    } else if (warp == 17) {
        // the run, by a scan over a head's blocks
        const int64_t total = a.head_units * c.n_kv, u0 = total * blockIdx.x / gridDim.x, u1 = total * (blockIdx.x + 1) / gridDim.x;
        const int g = (int)(u0 / a.head_units);
        const int64_t off = u0 - g * a.head_units;
        int64_t before = 0;  // units of the blocks before
        for (int b0 = 0; b0 < a.blocks; b0 += 32) {
            KpItem x;
            x.g = g, x.blk = b0 + lane, x.s = 0;
            int units = 0;
            if (x.blk < a.blocks) {
                x.in_run(a, 1);
                units = x.units();
            }
            int64_t end = units;
#pragma unroll
            for (int i = 1; i < 32; i <<= 1) {
                const int64_t v = __shfl_up_sync(0xffffffffu, end, i);
                if (lane >= i) end += v;
            }
            end += before;
            const unsigned found = __ballot_sync(0xffffffffu, end > off);
            if (found) {
                if (lane == __ffs(found) - 1) {
                    const int64_t at = g * a.head_units + end - units;  // the block's first unit
                    bars.g = g, bars.blk = x.blk, bars.s = (int)(at - u0), bars.len = (int)(u1 - u0);
                    x.s = bars.s;
                    x.in_run(a, bars.len);
                    const int w = x.mt() == 2 ? KP_UNITS : KP_UNITS1, ctas = (int)gridDim.x;
                    const bool cut = x.tile0 > 0 && x.n > 0;
                    bars.cut = KpCut{x.blk, g, cut ? kp_run_of(at + KP_UNITS_BLOCK, total, ctas) : -1,
                                     kp_run_of(at + KP_UNITS_BLOCK + (int64_t)(x.tiles - 1) * w, total, ctas)};
                }
                break;
            }
            before = __shfl_sync(0xffffffffu, end, 31);
        }
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = bars.tmem;
    KpItem it;
    it.g = bars.g, it.blk = bars.blk, it.s = bars.s;
    const int len = bars.len;
    // Every role runs through the items, and through them again if the first pass met a big scale: barriers and counters go on
    // as if these were further items, and all that was written is written anew
    bool second = false;
    auto again = [&]() {
        if (second) return false;
        kp_meet(true);
        second = bars.big && !bars.failed;
        it.g = bars.g, it.blk = bars.blk, it.s = bars.s;
        return second;
    };
    float *cs_smem = reinterpret_cast<float *>(smem + Cfg::CS);  // [KP_ROWS]
    pdl_wait();
    pdl_trigger();
    if (!a.whole && threadIdx.x == 17 * 32 && blockIdx.x > 0) {
        KpCut cut = bars.cut;
        const bool second = cut.first == (int)blockIdx.x - 1;
        if (!second) cut.first = -1;
        if (!a.by_item)
            a.cuts[blockIdx.x - 1] = cut;
        else if (second)
            a.cuts[cut.g * a.blocks + cut.blk] = cut;
    }

    if (warp < 8) {
        tc::more_registers<KP_REGS_SOFTMAX>();
        // ------------------------------------------------------------ the softmax: a thread per row
        const int m = warp >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + m * KP_N + lanes, to = tmem + 256 + m * HD + lanes;
        int nt = 0, items = 0;  // tiles and blocks before
        do {  // the passes
        for (; it.in_run_warp(a, len); it.next(a)) {
            if (it.n == 0 || m >= it.mt()) continue;
            KP_WAIT_WARP(bars.q_full[m], items & 1);
            float cs = cs_smem[m * KP_M + r];
            float &up = reinterpret_cast<float *>(smem + Cfg::UP)[m * KP_M + r];  // 2^kv4_far: cs and ref are the row's own over it
            up = 1.0f;
            const int t = a.pos0 + a.token(min(it.row0 + m * KP_M + r, it.row0 + it.n_rows - 1));  // the row's position
            const int row_lo = it.row0 + m * KP_M, row_hi = min(row_lo + KP_M, it.row0 + it.n_rows) - 1;
            // the tile's first and last position, and the last positions before their windows
            const int t_lo = kp_uniform(a.pos0 + a.token(row_lo)), t_hi = kp_uniform(a.pos0 + a.token(row_hi));
            const int w_lo = a.window > 0 ? t_lo - a.window : -1, w_hi = a.window > 0 ? t_hi - a.window : -1;
            if (lane == 0) bars.item[warp] = it;  // out of the registers while the tiles are worked on
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.q_empty[m]);
            float ref = -INFINITY, l = 0.0f;
            // which of the positions k0 .. k0 + 31 the row sees: those up to its own, of them the window's and the sinks
            auto sees32 = [&](int k0) {
                auto below = [](int x) { return (uint32_t)((1ull << min(max(x, 0), 32)) - 1); };
                return below(t + 1 - k0) & (a.window > 0 ? ~below(t - a.window + 1 - k0) | below(a.n_sink - k0) : ~0u);
            };
            // P of 32 columns of S against a reference (exponents s c + r), and its sum
            auto exps = [&](const uint32_t (&s)[32], uint32_t *p, uint64_t c2, uint64_t r2, uint64_t (&sum)[2], uint32_t see, auto masked) {
                // by stages over all 32: a group at a time would wait for each result
                uint64_t x[16];
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    uint32_t v[2] = {s[2 * i], s[2 * i + 1]};
                    if constexpr (decltype(masked)::value) {
#pragma unroll
                        for (int u = 0; u < 2; u++)
                            if (!(see & (1u << (2 * i + u)))) v[u] = 0xff800000u;  // -inf
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
            int left = it.n, k_tile = it.seen.tile(it.tile0) * KP_N;
            int sinks = it.seen.head - it.tile0;  // tiles to the last of the sinks'
            const int k_body = it.seen.body * KP_N;
            bool fresh = true;  // there is a row without a reference
#pragma unroll 1
            for (; left > 0; left--, nt++) {
                // settled before the wait, so that it is not on the way from S to P
                const bool whole = k_tile + KP_N - 1 <= t_lo && (k_tile > w_hi || k_tile + KP_N <= a.n_sink);
                KP_WAIT_WARP(bars.s_full[m], nt & 1);
                tc::fence_after();
                tc::ld32(ts, s0);
                // In halves of 64 positions, so that the first one's product runs beside the second's exps; half of the
                // next 64 columns is read while the second half of these is worked on
#pragma unroll 1
                for (int hf = 0; hf < 2; hf++) {
                    const int k0 = k_tile + 64 * hf;
                    const uint32_t th = ts + 64 * hf;
                    tc::ld32(th + 32, s1);
                    tc::wait_ld(s0);
                    tc::wait_ld(s1);
                    if (!whole && (k0 > t_hi || (k0 + 63 <= w_lo && k0 >= a.n_sink))) {  // no row sees any
#pragma unroll
                        for (int i = 0; i < 32; i++) p[i] = 0;
                        if (!hf) tc::ld32(ts + 64, s0);
                    } else {
                        bool raise = fresh;
                        float sum;
#pragma unroll 1
                        for (int again = 0;; again = 1) {
                            if (raise) {
                                if (again) {
                                    tc::wait_ld(s0);
                                    tc::ld32(th, s0);
                                    tc::ld32(th + 32, s1);
                                    tc::wait_ld(s0);
                                    tc::wait_ld(s1);
                                }
                                float mx = -INFINITY;
                                const uint32_t see0 = sees32(k0), see1 = sees32(k0 + 32);
#pragma unroll
                                for (int i = 0; i < 32; i++) {
                                    mx = fmaxf(mx, see0 & (1u << i) ? __uint_as_float(s0[i]) : -INFINITY);
                                    mx = fmaxf(mx, see1 & (1u << i) ? __uint_as_float(s1[i]) : -INFINITY);
                                }
                                cs *= up, ref *= up;
                                float next = fmaxf(ref, mx * cs);
                                const int far = kv4_far(next);
                                const float down = kv4_pow2(-far);
                                cs *= down, next *= down, up = kv4_pow2(far);
                                const float f = ref == -INFINITY ? 0.0f : kv4_exp2(ref * down - next);
                                ref = next;
                                l *= f;
                                if (hf) {  // the first half's product has to be in O
                                    KP_WAIT_WARP(bars.o_half[m], nt & 1);
                                    tc::fence_after();
                                }
                                if (left < bars.item[warp].n || hf) {
#pragma unroll 1
                                    for (int ch = 0; ch < HD; ch += 32) {
                                        tc::ld32(to + ch, p);
                                        tc::wait_ld(p);
#pragma unroll
                                        for (int i = 0; i < 32; i++) p[i] = __float_as_uint(__uint_as_float(p[i]) * f);
                                        tc::st32(to + ch, p);
                                    }
                                }
                            }
                            const float neg_ref = KP_BIAS - (ref == -INFINITY ? 0.0f : ref);
                            const uint64_t c2 = tc::pair(cs, cs), r2 = tc::pair(neg_ref, neg_ref);
                            uint64_t sums[2] = {0, 0};
                            if (whole)
                                exps(s0, p, c2, r2, sums, ~0u, KpNo{});
                            else
                                exps(s0, p, c2, r2, sums, sees32(k0), KpYes{});
                            if (!hf) tc::ld32(ts + 64, s0);
                            if (whole)
                                exps(s1, p + 16, c2, r2, sums, ~0u, KpNo{});
                            else
                                exps(s1, p + 16, c2, r2, sums, sees32(k0 + 32), KpYes{});
                            const float2 x = tc::unpair(tc::add2(sums[0], sums[1]));
                            sum = x.x + x.y;
                            if (raise) break;
                            raise = __any_sync(0xffffffffu, sum > KP_MOST);
                            if (!raise) break;
                        }
                        l += sum;
                        if (fresh) fresh = __any_sync(0xffffffffu, ref == -INFINITY);
                    }
                    tc::st32(th, p);
                    tc::wait_st();
                    tc::fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bars.p_full[m][hf]);
                }
                k_tile = --sinks == 0 ? k_body : k_tile + KP_N;
            }
            // ---- the rows' results
            it = bars.item[warp];
            const float inv = l == 0.0f ? 0.0f : (second ? KP_BIG : 1.0f) / l;
            const int row = row_lo + r;
            float *part = nullptr;
            if (!it.uncut()) {  // O as it is, rows side by side
                float *piece = a.part + (2 * (int64_t)blockIdx.x + (it.tile0 > 0 ? 0 : 1)) * Cfg::PART;
                part = piece + (m * KP_M + r) * 4;
                float *stats = piece + KP_ROWS * HD + m * KP_M + r;
                // times KP_BIG, by its weight
                if (row <= row_hi) stats[0] = ref * up + (second ? KP_BIG_LOG2 : 0.0f), stats[KP_ROWS] = second ? l / KP_BIG : l;
            }
            const int tok = a.token(row);
            const unsigned long long out =
                reinterpret_cast<unsigned long long>(reinterpret_cast<T *>(a.out) + (int64_t)tok * a.out_ld +
                                                     (int64_t)(it.g * a.group + row - tok * a.group) * HD);
            KP_WAIT_WARP(bars.o_full[m], items & 1);
            items++;
            tc::fence_after();
#pragma unroll 1
            for (int ch = 0; ch < HD; ch += 32) {
                uint32_t o[32];
                tc::ld32(to + ch, o);
                tc::wait_ld(o);
                if (part) {
                    if (row <= row_hi) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            *reinterpret_cast<uint4 *>(part + (ch + i) * KP_ROWS) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                    }
                } else {
                    // Column 2e of 8 is value e, column 2e + 1 value 4 + e.  Four lanes exchange 16-byte pieces so that each
                    // store of theirs fills 64 bytes of one row.
                    uint32_t y[sizeof(T) == 2 ? 16 : 32];
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        float x[8];
#pragma unroll
                        for (int v = 0; v < 4; v++)
                            x[v] = __uint_as_float(o[i + 2 * v]) * inv, x[4 + v] = __uint_as_float(o[i + 2 * v + 1]) * inv;
#pragma unroll
                        for (int v = 0; v < 8; v++) {
                            if constexpr (sizeof(T) == 2) {
                                if (v & 1) y[(i + v) / 2] = kv4_pack_bf2(x[v - 1], x[v]);
                            } else {
                                y[i + v] = __float_as_uint(x[v]);
                            }
                        }
                    }
#pragma unroll
                    for (int q = 0; q < (sizeof(T) == 2 ? 16 : 32); q += 16) {
                        uint32_t *z = y + q;  // pieces z[4 i ..] of this row, then piece lane & 3 of rows i
#pragma unroll
                        for (int bit = 1; bit < 4; bit <<= 1) {
                            const bool up = lane & bit;
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                if (i & bit) continue;
#pragma unroll
                                for (int e = 0; e < 4; e++) {
                                    uint32_t &lo = z[4 * i + e], &hi = z[4 * (i | bit) + e];
                                    const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? lo : hi, bit);
                                    (up ? lo : hi) = got;
                                }
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            char *dst = reinterpret_cast<char *>(__shfl_sync(0xffffffffu, out, (lane & ~3) | i)) +
                                        ch * sizeof(T) + q * 4 + 16 * (lane & 3);
                            if ((row & ~3) + i <= row_hi)
                                *reinterpret_cast<uint4 *>(dst) = make_uint4(z[4 * i], z[4 * i + 1], z[4 * i + 2], z[4 * i + 3]);
                        }
                    }
                }
            }
            tc::fence_before();
        }
        } while (again());
    } else if (warp < 16) {
        tc::fewer_registers<KP_REGS_DEQUANT>();
        // ------------------------------------------------------------ dequantise: a thread per position
        const int r = threadIdx.x & 127;
        const bool is_v = warp >= 12;
        const uint32_t smem0 = smem_u32(smem);
        const int m = is_v;  // the Q tile that this group loads: before its first tile of all, later after a block's first tile
        int nt = 0, items = 0;
        do {
        for (; it.in_run_warp(a, len); it.next(a)) {
            if (it.n == 0) continue;
            const int q_at = nt ? 1 : 0;
#pragma unroll 1
            for (int j = 0; j < it.n || j <= q_at; j++) {
                const bool load_q = j == q_at && m < it.mt();
                const uint32_t q_tile = smem0 + Cfg::Q + m * Cfg::TILE;  // chunk c of row r at c ^ (r & 7)
                const int my_row = min(it.row0 + m * KP_M + r, it.row0 + it.n_rows - 1), tok = a.token(my_row);
                const T *my_q = reinterpret_cast<const T *>(a.q) + (int64_t)tok * a.q_ld +
                                (int64_t)(it.g * a.group + my_row - tok * a.group) * HD;
                constexpr int CH = HD / 8;
                if (load_q) {
                    if (items > 0) KP_WAIT_WARP(bars.q_empty[m], (items - 1) & 1);
                    if constexpr (sizeof(T) == 2) {  // the warp's 32 rows in flight, while a tile is dequantised
#pragma unroll 4
                        for (int i = 0; i < 32; i += 32 / CH) {
                            const int src = i + lane / CH, ch = lane % CH, rr = (warp & 3) * 32 + src;
                            const T *p = reinterpret_cast<const T *>(__shfl_sync(0xffffffffu, (unsigned long long)my_q, src)) + 8 * ch;
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                                             q_tile + (ch >> 3) * Cfg::HALF + rr * 128 + (((ch & 7) ^ (rr & 7)) << 4)),
                                         "l"(p)
                                         : "memory");
                        }
                        asm volatile("cp.async.commit_group;" ::: "memory");
                    }
                }
                if (j < it.n) {
                    const int i = 2 * nt + is_v, slot = nt & 1, rs = i % KP_RAW;
                    // 16-byte chunk c of row r lies at chunk c ^ (r & 7), so at `dst` ^ 16 c
                    const uint32_t dst = smem0 + (is_v ? Cfg::V : Cfg::K) + slot * Cfg::TILE + r * 128 + (r & 7) * 16;
                    const uint32_t raw = smem0 + Cfg::R + rs * Cfg::RAW, codes = raw + r * (HD / 2) + 16 * kv4_turn<HD>(r);
                    KP_WAIT_WARP(bars.raw_full[is_v][rs], (nt / KP_RAW) & 1);
                    if (nt >= 2) KP_WAIT_WARP(is_v ? bars.v_empty[slot] : bars.k_empty[slot], ((nt >> 1) - 1) & 1);
                    const int pos = it.seen.tile(it.tile0 + j) * KP_N + r;
                    const bool seen = it.seen.sees(pos, a.n_sink);  // a row that no query sees may hold anything
                    uint32_t sc[NB / 2], top = 0;
#pragma unroll
                    for (int b = 0; b < NB / 2; b++) {
                        sc[b] = tc::lds32(raw + Cfg::CODES + (r * NB + 2 * b) * 2);
                        if (!seen) sc[b] = 0;
                        top |= (sc[b] & 0x70007000u) + 0x10001000u;
                    }
                    if (second) {
#pragma unroll
                        for (int b = 0; b < NB / 2; b++) {
                            const __half2 most = __float2half2_rn(65504.0f);
                            __half2 h;
                            memcpy(&h, &sc[b], 4);
                            h = __hmax2(__hmin2(h, most), __hneg2(most));  // also keeps a NaN out
                            h = __hmul2(h, __float2half2_rn(1.0f / KP_BIG));
                            memcpy(&sc[b], &h, 4);
                        }
                    } else if (top & 0x80008000u) {  // 2^13 (bits 0x7000) and more
                        bars.big = 1;
                    }
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        const uint4 w = tc::lds128(codes ^ (16 * b));
                        __half2 d;
                        const uint32_t dd = __byte_perm(sc[b / 2], 0, b & 1 ? 0x3232 : 0x1010);
                        memcpy(&d, &dd, 4);
                        const uint32_t to = dst + (b >> 1) * Cfg::HALF;
                        const int c0 = (b & 1) * 4;
                        tc::sts128(to ^ (16 * (c0 + 0)), kp_word(w.x, d));
                        tc::sts128(to ^ (16 * (c0 + 1)), kp_word(w.y, d));
                        tc::sts128(to ^ (16 * (c0 + 2)), kp_word(w.z, d));
                        tc::sts128(to ^ (16 * (c0 + 3)), kp_word(w.w, d));
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(&bars.raw_empty[rs]);
                        mbar_arrive(is_v ? &bars.v_full[slot] : &bars.k_full[slot]);
                    }
                    nt++;
                }
                if (load_q) {
                    // A thread per row, scaled in place (f32 rows are read twice)
                    const uint32_t q_row = q_tile + r * 128 + (r & 7) * 16;
                    auto chunk = [&](int ch) { return (q_row + (ch >> 3) * Cfg::HALF) ^ ((ch & 7) * 16); };
                    float top = 0.0f;
                    if constexpr (sizeof(T) == 2) {
                        asm volatile("cp.async.wait_group 0;" ::: "memory");
                        __syncwarp();
#pragma unroll 4
                        for (int ch = 0; ch < CH; ch++) {
                            const uint4 u = tc::lds128(chunk(ch));
                            // magnitudes of bf16 order as their bits
                            const uint32_t h = __vmaxu2(__vmaxu2(u.x & 0x7fff7fffu, u.y & 0x7fff7fffu),
                                                        __vmaxu2(u.z & 0x7fff7fffu, u.w & 0x7fff7fffu));
                            top = fmaxf(top, fmaxf(__uint_as_float(h << 16), __uint_as_float(h & 0xffff0000u)));
                        }
                    } else {
#pragma unroll 4
                        for (int ch = 0; ch < CH; ch++) {
                            float x[8];
                            kv4_load_row(my_q + 8 * ch, x);
#pragma unroll
                            for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[e]));
                        }
                    }
                    // 2^e * top in [2^5, 2^6), or below where top < 2^-121: exact for bf16 values down to 2^-22 of the largest
                    const int e = top > 0.0f && top <= FLT_MAX ? min(5 + 127 - (int)(__float_as_uint(top) >> 23), 126) : 0;
                    const float up = kv4_pow2(e);
#pragma unroll 4
                    for (int ch = 0; ch < CH; ch++) {
                        float x[8];
                        if constexpr (sizeof(T) == 2) {
                            const uint4 u = tc::lds128(chunk(ch));
                            kv4_bf2(u.x, x[0], x[1]), kv4_bf2(u.y, x[2], x[3]), kv4_bf2(u.z, x[4], x[5]), kv4_bf2(u.w, x[6], x[7]);
                        } else {
                            kv4_load_row(my_q + 8 * ch, x);
                        }
#pragma unroll
                        for (int v = 0; v < 8; v++) x[v] *= up;
                        tc::sts128(chunk(ch), make_uint4(kv4_half2(x[0], x[4]), kv4_half2(x[1], x[5]), kv4_half2(x[2], x[6]),
                                                         kv4_half2(x[3], x[7])));
                    }
                    // log2 score of an accumulator's 1
                    cs_smem[m * KP_M + r] = kv4_factor(a.scale * 1.4426950408889634f * kv4_pow2(-e) * (second ? KP_BIG : 1.0f));
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bars.q_full[m]);
                    items++;
                }
            }
        }
        } while (again());
    } else {
        tc::fewer_registers<KP_REGS_ISSUE>();
        if (warp == 16) {
            // -------------------------------------------------------- the MMAs
            constexpr uint32_t id_qk = tc::idesc(KP_M, KP_N, false), id_pv = tc::idesc(KP_M, HD, true);
            const uint32_t q_lo = tc::desc_lo(smem_u32(smem + Cfg::Q), 16), k_lo = tc::desc_lo(smem_u32(smem + Cfg::K), 16),
                           v_lo = tc::desc_lo(smem_u32(smem + Cfg::V), Cfg::HALF);
            // S of tile nt, and with the last of m: K's slot is free, with a block's last: Q too
            auto qk = [&](int m, int nt, bool k_free, bool q_free) {
                const uint32_t a_lo = q_lo + m * (Cfg::TILE >> 4), b_lo = k_lo + (nt & 1) * (Cfg::TILE >> 4);
                if (tc::elect()) {
#pragma unroll
                    for (int k = 0; k < HD / 16; k++) {
                        const uint32_t off = ((k >> 2) * Cfg::HALF + (k & 3) * 32) >> 4;
                        tc::mma_ss(tmem + m * KP_N, a_lo + off, tc::DESC_HI, b_lo + off, tc::DESC_HI, id_qk, k > 0);
                    }
                    tc::commit(&bars.s_full[m]);
                    if (k_free) tc::commit(&bars.k_empty[nt & 1]);
                    if (q_free) tc::commit(&bars.q_empty[m]);
                }
                __syncwarp();
            };
            auto pv = [&](int m, int nt, int hf, bool first, bool v_free, bool last) {
                const uint32_t b_lo = v_lo + (nt & 1) * (Cfg::TILE >> 4) + hf * (64 * 128 >> 4);
                if (tc::elect()) {
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        tc::mma_ts(tmem + 256 + m * HD, tmem + m * KP_N + 64 * hf + 8 * k, b_lo + k * (2048 >> 4), tc::DESC_HI,
                                   id_pv, k > 0 || hf || !first);
                    if (hf == 0) {
                        tc::commit(&bars.o_half[m]);
                    } else {
                        if (v_free) tc::commit(&bars.v_empty[nt & 1]);
                        if (last) tc::commit(&bars.o_full[m]);
                    }
                }
                __syncwarp();
            };
            // One step a tile: its products with V, and S of the tile after it, which may be the next block's
            auto skip_empty = [&]() {  // to a block with tiles in the run, if there is one
                while (it.in_run_warp(a, len)) {
                    if (it.n > 0) return true;
                    it.next(a);
                }
                return false;
            };
            int nt = -1, pt[2] = {0, 0}, qt[2] = {0, 0};  // tiles; tiles and blocks of A and of B
            do {
            bool more = skip_empty();
            int j = -1, n = more ? it.n : 0, mt = 0;  // the tile of the products; -1: none yet
            while (more) {
                // the tile after (j, n, mt)
                int nj = j + 1, nn = n, nmt = mt;
                if (j < 0) {
                    nmt = it.mt();
                } else if (nj == n) {
                    it.next(a);
                    more = skip_empty();
                    if (more) nj = 0, nn = it.n, nmt = it.mt();
                }
                if (j >= 0) KP_WAIT_WARP(bars.v_full[nt & 1], (nt >> 1) & 1);
                for (int m = 0; m < 2; m++) {
                    if (j >= 0 && m < mt) {
                        for (int hf = 0; hf < 2; hf++) {
                            KP_WAIT_WARP(bars.p_full[m][hf], pt[m] & 1);
                            tc::fence_after();
                            pv(m, nt, hf, j == 0, m == mt - 1, j + 1 == n);
                        }
                        pt[m]++;
                    }
                    if (more && m < nmt) {
                        if (m == 0) KP_WAIT_WARP(bars.k_full[(nt + 1) & 1], ((nt + 1) >> 1) & 1);
                        if (nj == 0) {
                            KP_WAIT_WARP(bars.q_full[m], qt[m] & 1);
                            qt[m]++;
                        }
                        tc::fence_after();
                        qk(m, nt + 1, m == nmt - 1, nj + 1 == nn);
                    }
                }
                nt++;
                j = nj, n = nn, mt = nmt;
            }
            if (nt >= 0) nt--;  // the last tile again
            } while (again());
        } else if (warp == 17) {
        // ------------------------------------------------------------ raw tiles by bulk copies
        int i = 0;  // raw tiles before
        do {
        if (lane == 0) {
            bool ok = true;
            for (; ok && it.in_run(a, len); it.next(a)) {
                const int64_t head = ((int64_t)a.seq * c.n_kv + it.g) * c.n_ctx;
                if (a.by_item && it.uncut()) a.cuts[it.g * a.blocks + it.blk] = KpCut{it.blk, it.g, -1, -1};
                for (int j = 0; j < 2 * it.n; j++, i++) {
                    const int rs = i % KP_RAW;
                    if (i >= KP_RAW && !mbar_wait_bounded(&bars.raw_empty[rs], ((i / KP_RAW) - 1) & 1)) {
                        latch_error(a.err, TMOE_DEV_ERR_TIMEOUT);
                        ok = false, bars.failed = 1;
                        break;
                    }
                    const int p0 = it.seen.tile(it.tile0 + (j >> 1)) * KP_N;
                    const int np = min(KP_N, c.n_ctx - p0);  // the cache may end inside the last tile (at 64)
                    uint8_t *dst = smem + Cfg::R + rs * Cfg::RAW;
                    uint64_t *full = &bars.raw_full[j & 1][rs];
                    mbar_arrive_expect_tx(full, (uint32_t)(np * (HD / 2 + NB * 2)));
                    bulk_g2s(dst, (j & 1 ? c.vc : c.kc) + (head + p0) * (HD / 2), (uint32_t)(np * (HD / 2)), full);
                    bulk_g2s(dst + Cfg::CODES, (j & 1 ? c.vs : c.ks) + (head + p0) * NB, (uint32_t)(np * NB * 2), full);
                }
            }
            // whatever became of their readers, the CTA does not end before its copies
            for (int k = max(i - KP_RAW, 0); k < i; k++)
                mbar_wait_bounded(&bars.raw_full[k & 1][k % KP_RAW], ((k >> 1) / KP_RAW) & 1);
        }
        __syncwarp();
        } while (again());
        } else {
            kp_meet(false);
        }
    }
done:
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
    tc::fence_before();
    __syncthreads();
    if (warp == 16) {
        tc::fence_after();
        tc::dealloc(tmem, 512);
    }
}

// The pieces of a block that was cut: a thread per row and 8 values, and of those pieces every LISTS-th.  A block
// here has KP_ROWS / LISTS rows.  Few blocks of many pieces take 4 lists (33 tokens at 20000, 8 blocks in some 150 pieces: 7 us from HBM,
// with one 16); else a block has two pieces, mostly, and they are one thread's.
template <int HD, typename T, int LISTS>
__global__ void __launch_bounds__(KP_ROWS) kv4_join_kernel(const float *__restrict__ part, const KpCut *__restrict__ cuts,
                                                           T *__restrict__ out, int64_t out_ld, int rows, int G) {
    constexpr int DEEP = LISTS > 1 ? 6 : 2, R = KP_ROWS / LISTS;  // pieces in flight; rows
    __shared__ float sums[LISTS > 1 ? LISTS - 1 : 1][10][R];
    pdl_wait();
    pdl_trigger();
    const int g8 = blockIdx.x % (HD / 8), rb = blockIdx.x / (HD / 8) % LISTS;
    const KpCut cut = cuts[blockIdx.x / (HD / 8 * LISTS)];
    if (cut.first < 0) return;
    const int mine = threadIdx.x % R, list = threadIdx.x / R, r_blk = rb * R + mine;
    const int row = cut.blk * KP_ROWS + r_blk, g = cut.g, pieces = cut.last - cut.first + 1;
    constexpr int64_t STEP = 2 * Kv4PrefillCfg<HD>::PART;
    // the first run's tail, then the others' heads
    const float *p = part + cut.first * STEP;
    const float *stats = p + KP_ROWS * HD + r_blk;
    const float4 *o = reinterpret_cast<const float4 *>(p) + 2 * g8 * KP_ROWS + r_blk;
    float top = -INFINITY, L = 0.0f, x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 1
    for (int s0 = list; s0 < pieces && row < rows; s0 += DEEP * LISTS) {
        float r[DEEP], l[DEEP];
        float4 y[DEEP][2];
#pragma unroll
        for (int u = 0; u < DEEP; u++) {
            const int s = s0 + u * LISTS;
            r[u] = -INFINITY, l[u] = 0.0f, y[u][0] = y[u][1] = make_float4(0, 0, 0, 0);
            if (s < pieces) {
                const int64_t at = s * STEP + (s ? 0 : STEP / 2);
                r[u] = __ldcg(stats + at), l[u] = __ldcg(stats + at + KP_ROWS);
                y[u][0] = __ldcg(o + at / 4), y[u][1] = __ldcg(o + at / 4 + KP_ROWS);
            }
        }
        float next = top;
#pragma unroll
        for (int u = 0; u < DEEP; u++) next = fmaxf(next, r[u]);
        const float f = top == -INFINITY ? 1.0f : kv4_exp2(top - next);
        top = next, L *= f;
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] *= f;
#pragma unroll
        for (int u = 0; u < DEEP; u++) {
            const float w = r[u] == -INFINITY ? 0.0f : kv4_exp2(r[u] - top);  // without a reference nothing was seen
            L += w * l[u];
            // column 2e of a chunk is value e, column 2e + 1 value 4 + e
            x[0] += w * y[u][0].x, x[4] += w * y[u][0].y, x[1] += w * y[u][0].z, x[5] += w * y[u][0].w;
            x[2] += w * y[u][1].x, x[6] += w * y[u][1].y, x[3] += w * y[u][1].z, x[7] += w * y[u][1].w;
        }
    }
    if constexpr (LISTS > 1) {
        if (list > 0) {
            float (*z)[R] = sums[list - 1];
            z[0][mine] = top, z[1][mine] = L;
#pragma unroll
            for (int e = 0; e < 8; e++) z[2 + e][mine] = x[e];
        }
        __syncthreads();
        if (list > 0) return;
        float next = top;
#pragma unroll
        for (int i = 0; i < LISTS - 1; i++) next = fmaxf(next, sums[i][0][mine]);
        const float f = top == -INFINITY ? 0.0f : kv4_exp2(top - next);
        L *= f;
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] *= f;
#pragma unroll
        for (int i = 0; i < LISTS - 1; i++) {
            const float t = sums[i][0][mine], w = t == -INFINITY ? 0.0f : kv4_exp2(t - next);
            L += w * sums[i][1][mine];
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] += w * sums[i][2 + e][mine];
        }
    }
    if (row >= rows) return;
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] *= inv;
    kv4_store_row(out + (int64_t)(row / G) * out_ld + (int64_t)(g * G + row % G) * HD + 8 * g8, x);
}

// ------------------------------------------------------------------ launchers
size_t kv4_prefill_part_bytes(int sm_count) {
    return (size_t)sm_count * (sizeof(KpCut) + 2 * Kv4PrefillCfg<128>::PART * 4);
}

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
    const int64_t rows = (int64_t)x.n_tok * G, blocks = (rows + KP_ROWS - 1) / KP_ROWS;
    const int64_t items = blocks * c.n_kv;
    if (rows > (1 << 30) || items > (1 << 30)) return cudaErrorInvalidValue;
    // The work, and the most that a CTA gets if the blocks stay whole
    int64_t units = 0, most = 0, load[KP_MAX_CTAS] = {};
    const int turns = sm_count < items ? sm_count : (int)items;
    if (turns > KP_MAX_CTAS) return cudaErrorInvalidValue;
    for (int64_t i = 0, b = blocks - 1; b >= 0; b--) {
        const int64_t row = b * KP_ROWS, last = row + KP_ROWS < rows ? row + KP_ROWS - 1 : rows - 1;
        const int64_t cost = KP_UNITS_BLOCK + (int64_t)kp_seen(x.pos0, (int)(row / G), (int)(last / G), x.window, x.n_sink).tiles *
                                                  (last - row >= KP_M ? KP_UNITS : KP_UNITS1);
        units += cost;
        for (int g = 0; g < c.n_kv; g++, i++) {
            const int64_t turn = i / turns, at = i % turns;
            int64_t &l = load[turn & 1 ? turns - 1 - at : at];
            l += cost;
            if (l > most) most = l;
        }
    }
    const int64_t total = units * c.n_kv;
    // even runs: a CTA per SM, each with a block's cost and two tiles at least (so that every run has a tile)
    int64_t ctas = total / (KP_UNITS_BLOCK + 2 * KP_UNITS);
    ctas = ctas < 1 ? 1 : ctas < sm_count ? ctas : sm_count;
    if (total / ctas > (1 << 30)) return cudaErrorInvalidValue;
    Kv4PrefillArgs a;
    a.whole = most <= total / ctas + KP_UNITS_JOIN;
    if (a.whole) ctas = turns;
    a.q = x.q, a.out = x.out, a.q_ld = x.q_ld, a.out_ld = x.out_ld;
    a.seq = x.seq0, a.pos0 = x.pos0, a.n_tok = x.n_tok;
    a.window = x.window, a.n_sink = x.n_sink, a.scale = x.scale;
    a.group = G, a.group_inv = G > 1 ? ~0ull / G + 1 : 0, a.blocks = (int)blocks, a.n_kv = c.n_kv, a.head_units = units;
    a.cuts = reinterpret_cast<KpCut *>(part), a.part = part + sm_count * (sizeof(KpCut) / 4);
    a.by_item = items < ctas - 1;
    a.err = err;
    const cudaError_t e = launch_k(kv4_prefill_kernel<HD, T>, dim3((unsigned)ctas), dim3(KP_THREADS), (size_t)Cfg::SMEM, st, a, c);
    if (e != cudaSuccess || a.whole || ctas == 1) return e;
    return launch_k(a.by_item ? kv4_join_kernel<HD, T, 4> : kv4_join_kernel<HD, T, 1>,
                    dim3((unsigned)((a.by_item ? 4 * items : ctas - 1) * (HD / 8))), dim3(KP_ROWS), 0, st, (const float *)a.part,
                    (const KpCut *)a.cuts, (T *)x.out, x.out_ld, (int)rows, G);
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
