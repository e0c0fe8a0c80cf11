// The 4-bit KV cache (format: kv4.cuh): quantising rows into it, reading rows back, and the attention
// of single query tokens over it.
//   kv4_store_kernel   K and V rows -> codes and scales, at any (sequence, position) of each row
//   kv4_load_kernel    the same rows back as values
//   kv4_attn_kernel    one query token per sequence (a decode step), its K/V row quantised into the
//                      cache on the way; or a few tokens of one sequence
#include <algorithm>

#include "kernels.cuh"
#include "kv4.cuh"

namespace tmoe {

// ------------------------------------------------------------------ rows in and out
// Row i of a call: its sequence and position; false: no row.  A negative position means "no row" to
// the caller too; any other place outside the cache latches the device error.
struct Kv4RowArgs {
    void *k, *v;
    int64_t ld, n;
    const int32_t *seq, *pos;  // nullptr: seq0 (or row i of sequence i where it is negative), pos0 + i
    int seq0, pos0;
    Kv4Planes c;
    int *err;
};
__device__ __forceinline__ bool kv4_place(const Kv4RowArgs &a, int64_t i, int &s, int &p) {
    const int64_t ps = a.pos ? a.pos[i] : a.pos0 + i, sq = a.seq ? a.seq[i] : a.seq0 >= 0 ? a.seq0 : i;
    if (ps < 0) return false;
    if (ps >= a.c.n_ctx || sq < 0 || sq >= a.c.n_seq) {
        latch_error(a.err, TMOE_DEV_ERR_BADPOS);
        return false;
    }
    s = (int)sq, p = (int)ps;
    return true;
}

// Rows are independent and only moved once, so that what bounds it is the codes' instructions: 79% of the issue slots in a
// capture, 13% of DRAM.  A thread takes 16 values (a block is two threads, its extremes one shuffle each), so that a warp reads
// whole 128-byte lines; rows run fastest over the threads, so that a run of positions writes one contiguous piece of a
// head's plane.  8191 bf16 rows of 8 heads of 128, K and V: 12.5 us (43 MB, floor 6.6), f32 rows 13.0 (77 MB, 11.7); with 8
// values a thread and converted codes 20.6.
template <int HD, typename T>
__global__ void __launch_bounds__(256) kv4_store_kernel(const Kv4RowArgs a) {
    const Kv4Planes &c = a.c;
    constexpr int TPR = HD / 16, NB = HD / 32;
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t i = at / TPR;
    const int sub = (int)(at % TPR), b = sub >> 1;
    const int g = blockIdx.y >> 1;
    const bool is_v = blockIdx.y & 1;
    pdl_wait();
    pdl_trigger();
    float x[16];
#pragma unroll
    for (int j = 0; j < 16; j++) x[j] = 0.0f;
    int s = 0, p = 0;
    const bool ok = i < a.n && kv4_place(a, i, s, p);
    if (ok) kv4_load_row(reinterpret_cast<const T *>(is_v ? a.v : a.k) + i * a.ld + (int64_t)g * HD + 16 * sub, x);
    // NaN and infinity have the largest exponent: seldom there
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 16; j++) top = max(top, __float_as_uint(x[j]) & 0x7fffffffu);
    if (top >= 0x7f800000u) {
#pragma unroll
        for (int j = 0; j < 16; j++) x[j] = kv4_finite(x[j]);
    }
    float hi = x[0], lo = x[0];
#pragma unroll
    for (int j = 1; j < 16; j++) hi = fmaxf(hi, x[j]), lo = fminf(lo, x[j]);
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, 1));
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, 1));
    __half d;
    float inv;
    kv4_scale(hi, lo, d, inv);
    if (!ok) return;
    const int64_t row = ((int64_t)s * c.n_kv + g) * c.n_ctx + p;
    uint8_t *codes = (is_v ? c.vc : c.kc) + row * (HD / 2);
    *reinterpret_cast<uint2 *>(codes + 16 * (b ^ kv4_turn<HD>(p)) + 8 * (sub & 1)) =
        make_uint2(kv4_word<8>(x, inv), kv4_word<8>(x + 8, inv));
    if ((sub & 1) == 0) (is_v ? c.vs : c.ks)[row * NB + b] = d;
}

// A thread writes 8 values (16 bytes of bf16), so that a warp's stores are whole lines.  HBM-bound.  The same rows as f32: 14.4 us
// (77 MB, floor 11.7); two rows a thread 16.5, four 19.7.
template <int HD, typename T>
__global__ void __launch_bounds__(256) kv4_load_kernel(const Kv4RowArgs a) {
    const Kv4Planes &c = a.c;
    constexpr int TPR = HD / 8, NB = HD / 32;
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t i = at / TPR;
    const int sub = (int)(at % TPR), b = sub >> 2;
    const int g = blockIdx.y >> 1;
    const bool is_v = blockIdx.y & 1;
    pdl_wait();
    pdl_trigger();
    if (i >= a.n) return;
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    int s, p;
    if (kv4_place(a, i, s, p)) {
        const int64_t row = ((int64_t)s * c.n_kv + g) * c.n_ctx + p;
        const uint8_t *codes = (is_v ? c.vc : c.kc) + row * (HD / 2);
        const uint32_t w = *reinterpret_cast<const uint32_t *>(codes + 16 * (b ^ kv4_turn<HD>(p)) + 4 * (sub & 3));
        const float d = __half2float((is_v ? c.vs : c.ks)[row * NB + b]);
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = d * (__uint_as_float(0x4b000000u | ((w >> (4 * j)) & 15u)) - 8388616.0f);
    }
    kv4_store_row(reinterpret_cast<T *>(is_v ? a.v : a.k) + i * a.ld + (int64_t)g * HD + 8 * sub, x);
}

// ------------------------------------------------------------------ attention of single tokens
// For each query token and KV head: softmax(q K^T) V over the seen positions, up to 8 of the head's query
// heads together (more are further passes over the same rows, from L2).
//
// Bound: HBM (a cached position is read once, 4.5 bits a value).  At that rate an SM has about 390
// clocks for a 64-position tile of 128-wide K and V, 1560 issue slots, so the work per value has to be
// small:
//   - Codes meet the tensor cores as they are, as the 16-row operand of mma.sync m16n8k16 (f16 operands, f32
//     sums); the 8 heads are the 8 columns.  S^T = K Q^T: a 4-bit code under a mask is the f16 subnormal
//     c * 2^-24 (or 16 times that), so a word of 8 codes becomes four operand registers with four ANDs and one
//     shift.  The factor 16 is undone in Q.  A block's scale multiplies its own accumulator in f32: K
//     enters exactly.  The codes' -8 is a product of its own, scales x (-8 sum of q per block), on m16n8k8 (with
//     f32 queries it is taken from the codes, as for V: sums around 0 keep the scores' last bits).
//   - O^T += V^T P takes V as 1024 + c minus 1032 in f16 (here the -8 has to go before the product:
//     averaged over many positions, sum(P c) - 8 sum(P) would cancel), its scale on P.
//   - K's words through ldmatrix are the operand of two steps of 16 dimensions; V's 16-bit units (4 codes)
//     through ldmatrix.trans are, mask by mask, the operand's rows.  P takes one movmatrix per 8 positions.
//   - A head's reference moves only when a score exceeds it by more than 2^8, so that no tile waits for a
//     reduction over the warp.
// Precision: Q is scaled by a power of two per head into f16's upper range; bf16 queries then are exact.
// f32 queries, and P with them, are split into high + low f16 parts, in two products.  P times the V scale is
// held relative to the reference and to the largest V scale seen in the same block of 32 dimensions, so that neither small
// scales nor another block's large ones leave it in f16's subnormals.  For bf16 P is rounded to f16, and its product with the
// scale again (2^-11 relative each, below the output's own 2^-8).  A scale below 2^-14 of its block's largest loses last bits there.
//
// Work: the tiles of all (token, KV head, pass) are one list, cut into equal runs, one per CTA: ragged
// lengths, few sequences or many all load every SM the same.  A segment (one token, KV head and pass)
// costs a CTA about PART tiles' time to begin and to join, so that a segment counts that much more in
// the list; where the segments are few against the CTAs, each is instead padded to whole runs, and no
// CTA has more than one (the cheaper of the two by its longest run).  A warp takes every WARPS-th tile of a
// run, fetched by bulk copies into its own ring.  Runs that hold less than a segment leave partial sums in
// scratch; the CTA that arrives last there joins them, in run order (the same sums every call).
//
// Measured (32 heads, width 128, bf16; graph replay): 64 sequences of up to 32768 positions, 4 KV heads, 150 to 160 us by device,
// 4.8 to 5.1 TB/s; one of 131071, 8 KV heads, 40 us, 3.8 TB/s.  What is left there: the SMs get unequal shares of the bandwidth
// (their even runs end 138 .. 150 us), and a part's start and join are about 5 us.
constexpr int KA_HEADS = 8;
constexpr float KA_ROOM = 8.0f;  // how far (log2) a score may exceed its head's reference
constexpr float KA_BIAS = 6.0f;  // P times the V scale is held below 2^(KA_BIAS + KA_ROOM)

struct Kv4AttnArgs {
    const void *q, *k, *v;  // k == nullptr: the new rows are in the cache already
    void *out;
    int64_t q_ld, kv_ld, out_ld;
    const int32_t *pos;  // nullptr: token t at pos0 + t
    int pos0, seq0;      // seq0 >= 0: every token is of that sequence; else token t of sequence t
    int n_tok, n_head, window, n_sink;
    float scale;
    int *arrived;  // [grid] parts of the segment that starts in a run; zero between calls
    float *part;   // [grid][2][KA_HEADS][HD + 2]
    int *err;
};

template <int HD, bool PREC, bool SHORT>
struct Kv4AttnCfg {
    static constexpr int NB = HD / 32;
    static constexpr int TILE = 64;  // positions; in tiles of 32 all of the cases below took 5 to 25% longer
    // Warps of a CTA, tiles in a warp's ring, CTAs of an SM.  Per SM about 200 KB of ring and as many warps as registers allow;
    // which split is best was measured:
    //   width 128, bf16, 64 x 32768 / 1 x 131071: 12 x 2, one CTA 149 / 39.8 us; 8 x 3, one 160 / 41.6; 6 x 2, two 157 / 42.4
    //   width 128, f32, 4 x 4096: 8 x 3, one CTA 11.1 us; 12 x 2, one 13.3; 6 x 2, two 15.3
    //   width 64, 16 heads over 16, 24 x 5003: 6 x 4, two CTAs 32.3 us; 12 x 4, one 37.2; 8 x 6, one 38.5
    // (sequences here and below: of up to that many positions, the mean 0.62 of it)
    // SHORT: more segments than SMs, of 128 tiles at most each.  A CTA's start and join then come often, and run beside a second
    // CTA's tiles: width 128, bf16, 6 x 2, two CTAs against 12 x 2, one, in 64 sequences of 1024 / 4096 / 8192 / 16384 positions
    // 19.3 / 38.5 / 61.9 / 98.7 us against 21.4 / 41.8 / 61.9 / 96.1; f32, 4 x 3, two against 8 x 3, one, 21.3 / 50.1 / 83.9 / 137.0
    // against 22.7 / 53.7 / 84.2 / 137.9.
    static constexpr int WARPS = HD == 64 ? 6 : SHORT ? (PREC ? 4 : 6) : PREC ? 8 : 12, STAGES = HD == 64 ? 4 : PREC ? 3 : 2;
    static constexpr int CTAS = HD == 64 || SHORT ? 2 : 1;
    // In tiles, what a segment costs besides its own (f32's take longer): f32, 16 / 20 / 32 in 64 sequences of 8192 77.7 / 78.9 / 83.7
    // us, 16 of 2048 15.6 / 13.9 / 13.9; bf16, 12 / 20 / 32 / 48 in 32 of 4096 (window, 40 heads over 8) 44.3 / 44.0 / 42.4 / 43.4.
    static constexpr int PART = PREC ? 20 : 32;
    static constexpr int THREADS = 32 * WARPS;
    static constexpr int CODES = TILE * HD / 2, SCALES = TILE * NB * 2;
    static constexpr int STAGE = 2 * (CODES + SCALES);  // K codes, V codes, K scales, V scales
    static constexpr int VCODES = CODES, KSCALES = 2 * CODES, VSCALES = 2 * CODES + SCALES;
    static constexpr int RING = WARPS * STAGES * STAGE;
    static constexpr int SMEM = RING + WARPS * STAGES * 8 + 128;
    static_assert(WARPS * KA_HEADS * (HD + 2) * 4 <= RING, "the warps' sums are joined in the ring's space");
};

__device__ __forceinline__ void ka_ldsm(uint32_t addr, uint32_t &r0, uint32_t &r1, uint32_t &r2, uint32_t &r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
                 : "r"(addr));
}
__device__ __forceinline__ void ka_ldsm_t(uint32_t addr, uint32_t &r0, uint32_t &r1, uint32_t &r2, uint32_t &r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
                 : "r"(addr));
}
__device__ __forceinline__ uint32_t ka_transpose(uint32_t u) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(u));
    return r;
}
// d += a b
__device__ __forceinline__ void ka_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ka_mma8(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(b0));
}
__device__ __forceinline__ __half2 ka_h2(uint32_t u) {
    __half2 h;
    memcpy(&h, &u, 4);
    return h;
}
__device__ __forceinline__ uint32_t ka_u(__half2 h) {
    uint32_t u;
    memcpy(&u, &h, 4);
    return u;
}
__device__ __forceinline__ float2 ka_float2(uint32_t u) { return __half22float2(ka_h2(u)); }
// hi = f16(a, b), lo = f16 of what that leaves
__device__ __forceinline__ void ka_split(float a, float b, uint32_t &hi, uint32_t &lo) {
    hi = kv4_half2(a, b);
    const float2 f = ka_float2(hi);
    lo = kv4_half2(a - f.x, b - f.y);
}
// (u & mask | 1024) - off as f16 pairs
__device__ __forceinline__ uint32_t ka_codes(uint32_t u, uint32_t mask, __half2 off) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(u), "r"(mask), "r"(0x64006400u));  // (u & mask) | magic
    return ka_u(__hsub2(ka_h2(r), off));
}

template <int HD, typename T, bool SHORT>
__global__ void __launch_bounds__((Kv4AttnCfg<HD, sizeof(T) == 4, SHORT>::THREADS), (Kv4AttnCfg<HD, sizeof(T) == 4, SHORT>::CTAS))
    kv4_attn_kernel(const Kv4AttnArgs a, const Kv4Planes c) {
    constexpr bool PREC = sizeof(T) == 4;
    using Cfg = Kv4AttnCfg<HD, PREC, SHORT>;
    constexpr int PART = Cfg::PART;
    constexpr int NB = Cfg::NB, ST = Cfg::STAGES, RW = HD + 2, TILE = Cfg::TILE, HB = TILE / 16, WARPS = Cfg::WARPS;
    constexpr uint32_t M1 = 0x000f000fu, M16 = 0x00f000f0u;
    extern __shared__ __align__(128) uint8_t ka_smem[];
    uint64_t *bars = reinterpret_cast<uint64_t *>(ka_smem + Cfg::RING);
    __shared__ int sh_last;
    __shared__ float sh_up[Cfg::WARPS][KA_HEADS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gr = lane >> 2, t4 = lane & 3;
    const int G = a.n_head / c.n_kv, passes = (G + KA_HEADS - 1) / KA_HEADS, H = c.n_kv * passes;
    uint64_t *bar = bars + warp * ST;
    if (lane == 0)
        for (int s = 0; s < ST; s++) mbar_init(&bar[s], 1);
    fence_barrier_init();
    __syncwarp();  // a warp's barriers are its own
    pdl_wait();
    pdl_trigger();

    auto pos_of = [&](int t) -> int {  // -1: no query, -2: a place outside the cache
        const int64_t p = a.pos ? a.pos[t] : (int64_t)a.pos0 + t;
        if (p >= c.n_ctx) return -2;
        return p < 0 ? -1 : (int)p;
    };
    // The list: token t's segments, H of them (KV heads times passes), t ascending; below 2^31 entries by the
    // host's check.  Every warp works out the same: a lane takes `chunk` neighbouring tokens (one, up to 32).
    const int chunk = (a.n_tok + 31) / 32, lane_t0 = lane * chunk, lane_t1 = min(lane_t0 + chunk, a.n_tok);
    int p_first = -1, n_first = 0;  // of the lane's first token: its position, its tiles
    auto tiles_at = [&](int p) { return p < 0 ? 0 : Kv4Seen::of<TILE>(p, a.window, a.n_sink).tiles; };
    auto tiles_of = [&](int t) { return t == lane_t0 ? n_first : tiles_at(pos_of(t)); };
    int total = 0, live = 0;  // tiles and tokens with a query
    if (lane_t0 < lane_t1) p_first = pos_of(lane_t0), n_first = tiles_at(p_first);
#pragma unroll 1
    for (int t = lane_t0; t < lane_t1; t++) {
        const int n = tiles_of(t);
        total += n, live += n > 0;
    }
    total = __reduce_add_sync(0xffffffffu, total) * H;
    live = __reduce_add_sync(0xffffffffu, live);
    const bool idle = live < a.n_tok;
    live *= H;
    const int grid = gridDim.x;
    // runs of whole segments' pieces, a tile a warp at least; or runs over the list as it comes
    const int alone = live < grid ? max((total + grid - live - 1) / (grid - live), WARPS) : 0x7fffffff;
    const int across = (int)(((int64_t)total + (int64_t)live * PART + grid - 1) / grid);
    const bool pad = alone <= across;
    const int per = max(pad ? alone : across, 1);
    auto length = [&](int n) { return n == 0 ? 0 : pad ? (n + per - 1) / per * per : n + PART; };
    int entries = 0;  // of the lane's tokens
#pragma unroll 1
    for (int t = lane_t0; t < lane_t1; t++) entries += H * length(tiles_of(t));
    int before = entries;  // of the tokens before the lane's
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += up;
    }
    const int all = __shfl_sync(0xffffffffu, before, 31);
    before -= entries;
    // tokens without a query: zeros
    for (int t = blockIdx.x; idle && t < a.n_tok; t += gridDim.x) {
        const int p = pos_of(t);
        if (p >= 0) continue;
        if (p == -2 && threadIdx.x == 0) latch_error(a.err, TMOE_DEV_ERR_BADPOS);
        T *o = reinterpret_cast<T *>(a.out) + (int64_t)t * a.out_ld;
        const float z[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        for (int i = threadIdx.x; i < a.n_head * HD / 8; i += Cfg::THREADS) kv4_store_row(o + 8 * i, z);
    }
    // the ring: the next stage to fill and to read, and the phase of the latter
    int st_fill = 0, st_read = 0;
    uint32_t phase = 0;
    const uint32_t ring = smem_u32(ka_smem) + warp * ST * Cfg::STAGE;
    // where a lane reads in a stage: K and V rows as ldmatrix operands, scales of rows gr (K) and 2 t4 (V)
    uint32_t at_codes;
    if constexpr (HD == 128)  // 8 rows, a block per 8 lanes
        at_codes = (lane & 7) * 64 + 16 * ((lane >> 3) ^ kv4_turn<128>(lane & 7));
    else  // 16 rows: lanes 0..15 rows 0..7 of blocks 0, 1; lanes 16..31 rows 8..15
        at_codes = ((lane & 7) + 8 * (lane >> 4)) * 32 + 16 * (((lane >> 3) & 1) ^ kv4_turn<64>(lane & 7));
    const __half2 off1 = __float2half2_rn(1032.0f), off16 = __float2half2_rn(1152.0f);

    const int run = blockIdx.x, start = run * per, end = min(start + per, all);
    if (start >= end) return;
    // the token whose entries hold `start`, where they begin, the token's position
    int tok = 0, tok0 = 0, p_new = 0;
    {
        const bool mine = before <= start && start < before + entries;
        if (mine) {
            tok = lane_t0, tok0 = before, p_new = p_first;
#pragma unroll 1
            for (;;) {
                const int len = H * length(tiles_of(tok));
                if (start < tok0 + len) break;
                tok0 += len, tok++;
            }
            if (tok != lane_t0) p_new = pos_of(tok);
        }
        const int src = __ffs(__ballot_sync(0xffffffffu, mine)) - 1;
        tok = __shfl_sync(0xffffffffu, tok, src), tok0 = __shfl_sync(0xffffffffu, tok0, src);
        p_new = __shfl_sync(0xffffffffu, p_new, src);
    }
    int at = start;
    bool dead = false;  // a wait ran out: the warp fetches nothing more, as its barriers' phases may be open
    while (at < end) {
        if (p_new < 0) {
            p_new = pos_of(++tok);
            continue;
        }
        const Kv4Seen seen = Kv4Seen::of<TILE>(p_new, a.window, a.n_sink);
        const int len = length(seen.tiles), hc = (at - tok0) / len;
        const int seg0 = tok0 + hc * len, upto = min(end, seg0 + len);
        // the segment's tiles first .. first + n_part - 1, and whose runs hold the others
        int first, n_part, first_run, parts;
        if (pad) {
            parts = len / per, first_run = seg0 / per;
            const int i = run - first_run;
            const int each = seen.tiles / parts, more = seen.tiles - each * parts;
            first = i * each + min(i, more), n_part = each + (i < more);
        } else {
            // its tiles are the entries from seg0 + PART on
            first = max(at - seg0 - PART, 0);
            n_part = upto - seg0 - PART - first;
            first_run = (seg0 + PART) / per, parts = (seg0 + len - 1) / per - first_run + 1;
        }
        at = upto;
        const int t = tok, p_tok = p_new;
        if (at == tok0 + H * len) {
            tok0 = at, tok++;
            if (at < end) p_new = pos_of(tok);
        }
        if (n_part <= 0) continue;
        const int g = hc / passes, h0 = (hc % passes) * KA_HEADS;
        const int heads = min(G - h0, KA_HEADS);
        const int64_t row0 = ((int64_t)(a.seq0 >= 0 ? a.seq0 : t) * c.n_kv + g) * c.n_ctx;

        // ---- this warp's tiles: first + warp, first + warp + WARPS, ...  Lanes 0..3 copy a plane's piece each
        const int mine = n_part > warp && !dead ? (n_part - warp + WARPS - 1) / WARPS : 0;
        const uint8_t *src;
        uint32_t piece, dst;
        {
            const bool is_v = lane & 1, is_scale = lane & 2;
            piece = is_scale ? Cfg::SCALES : Cfg::CODES;
            dst = ring + (is_scale ? Cfg::KSCALES : 0) + (is_v ? piece : 0);
            src = (is_scale ? reinterpret_cast<const uint8_t *>(is_v ? c.vs : c.ks) : is_v ? c.vc : c.kc) +
                  row0 * (piece / TILE);
        }
        auto fill = [&](int j) {
            uint64_t *b = &bar[st_fill];
            if (lane == 0) mbar_arrive_expect_tx(b, Cfg::STAGE);
            if (lane < 4)
                asm volatile(
                    "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                        dst + st_fill * Cfg::STAGE),
                    "l"(src + (int64_t)seen.tile(first + warp + j * WARPS) * piece), "r"(piece), "r"(smem_u32(b))
                    : "memory");
            st_fill = st_fill + 1 == ST ? 0 : st_fill + 1;
        };
        int filled;
        auto fill_first = [&]() {
#pragma unroll 1
            for (filled = 0; filled < mine && filled < ST; filled++) fill(filled);
        };
        fill_first();

        // ---- Q operand: column gr is head gr of the pass; of block b the thread has dims 32 b + 8 t4 + 0..7, as
        // pairs (0, 4), (1, 5) / 16, (2, 6), (3, 7) / 16, matching the codes' order in a word
        uint32_t qh[NB][4], ql[PREC ? NB : 1][4];
        uint32_t q_sums;      // -8 * 2^-24 * sum of q of blocks 2 (t4 & 1), 2 (t4 & 1) + 1; t4 < 2 high parts, else low
        float to_log2[2];     // of heads 2 t4, 2 t4 + 1: log2 score of an accumulator's 1
        {
            float x[NB][8];
            float top = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; b++) {
#pragma unroll
                for (int i = 0; i < 8; i++) x[b][i] = 0.0f;
                if (gr < heads)
                    kv4_load_row(reinterpret_cast<const T *>(a.q) + (int64_t)t * a.q_ld +
                                     (int64_t)(g * G + h0 + gr) * HD + 32 * b + 8 * t4, x[b]);
#pragma unroll
                for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf(x[b][i]));
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // 2^e * top in [2^13, 2^14); two factors, as 2^e alone may not be a float
            const int e = top > 0.0f && top <= FLT_MAX ? 13 - ilogbf(top) : 0;
            const int e1 = e / 2, e2 = e - e1;
            const float up1 = kv4_pow2(e1), up2 = kv4_pow2(e2);
            constexpr int HALF_UNIT = PREC ? 0 : 12;  // codes count 1 with f32, 2^-24 with bf16
            const float c_gr = kv4_factor(a.scale * 1.4426950408889634f * kv4_pow2(HALF_UNIT - e1) * kv4_pow2(HALF_UNIT - e2));
            to_log2[0] = __shfl_sync(0xffffffffu, c_gr, 8 * t4);
            to_log2[1] = __shfl_sync(0xffffffffu, c_gr, 8 * t4 + 4);
            uint32_t sums[2] = {0, 0};  // [low]: of this lane's two blocks
            float pair = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                float z[8], sq = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) z[i] = x[b][i] * up1 * up2;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const __half2 r = __float2half2_rn(i & 1 ? 0.0625f : 1.0f);
                    float2 f;
                    if constexpr (PREC) {
                        ka_split(z[i], z[i + 4], qh[b][i], ql[b][i]);
                        f = ka_float2(ql[b][i]);
                        sq += f.x + f.y;
                        ql[b][i] = ka_u(__hmul2(ka_h2(ql[b][i]), r));
                    } else {
                        qh[b][i] = kv4_half2(z[i], z[i + 4]);
                    }
                    f = ka_float2(qh[b][i]);
                    sq += f.x + f.y;
                    qh[b][i] = ka_u(__hmul2(ka_h2(qh[b][i]), r));
                }
                sq += __shfl_xor_sync(0xffffffffu, sq, 1);
                sq += __shfl_xor_sync(0xffffffffu, sq, 2);
                sq *= -0x1p-21f;
                if (b & 1) {
                    if ((t4 & 1) == b / 2) ka_split(pair, sq, sums[0], sums[1]);
                } else {
                    pair = sq;
                }
            }
            q_sums = t4 < 2 ? sums[0] : sums[1];
        }
        bool held = false;  // the second time, for references past 2^24 (kv4_far)
    tiles:
        float o[NB][2][4];  // [block][values 0, 1 or 2, 3 of 4 gr ..]: rows (value, head 2 t4 + {0, 1})
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 2; i++) o[b][i][0] = o[b][i][1] = o[b][i][2] = o[b][i][3] = 0.0f;
        // of heads 2 t4 + {0, 1}: the reference, the sum over this thread's positions
        float ref[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
        // Of each block of 32 values, a pair of them a word: the f16 power of two that takes every V scale seen below 1.
        // O is held times it
        uint32_t room[NB / 2];
#pragma unroll
        for (int b = 0; b < NB / 2; b++) room[b] = 0x74007400u;  // 2^14
        auto room_of = [&](int b) {
            const float2 r = ka_float2(room[b / 2]);
            return b & 1 ? r.y : r.x;
        };

        for (int j = 0; j < filled; j++) {
            if (!__all_sync(0xffffffffu, mbar_wait_bounded(&bar[st_read], phase))) {
                if (lane == 0) latch_error(a.err, TMOE_DEV_ERR_TIMEOUT);
                dead = true;  // no more fills; the loop goes on to wait for those in flight
            }
            const uint32_t stage = ring + st_read * Cfg::STAGE;
            uint8_t *const stage_p = ka_smem + (stage - smem_u32(ka_smem));
            st_read++;
            if (st_read == ST) st_read = 0, phase ^= 1;
            const int p0 = seen.tile(first + warp + j * WARPS) * TILE;
            const bool whole = seen.whole(p0, TILE, a.n_sink), newest = p0 + TILE > p_tok;
            if (!dead) {
                if (!whole || newest) {
                    uint8_t *ks = stage_p + Cfg::KSCALES, *vs = stage_p + Cfg::VSCALES;
                    if (a.k && newest) {
                        // the new row: quantised into the tile, and (one pass only) into the cache
                        constexpr int LANES = HD / 4;
                        const int r = p_tok % TILE, b = lane >> 3;
#pragma unroll 1
                        for (int kv = 0; kv < 2; kv++) {
                            float x[4] = {0, 0, 0, 0};
                            if (lane < LANES)
                                kv4_load_row(reinterpret_cast<const T *>(kv ? a.v : a.k) + (int64_t)t * a.kv_ld +
                                                 g * HD + 4 * lane, x);
                            float hi = -FLT_MAX, lo = FLT_MAX;
#pragma unroll
                            for (int i = 0; i < 4; i++)
                                x[i] = kv4_finite(x[i]), hi = fmaxf(hi, x[i]), lo = fminf(lo, x[i]);
#pragma unroll
                            for (int m = 1; m <= 4; m <<= 1) {
                                hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, m));
                                lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, m));
                            }
                            __half d;
                            float inv;
                            kv4_scale(hi, lo, d, inv);
                            const uint32_t w = kv4_word<4>(x, inv);
                            if (lane < LANES) {
                                const int byte = 16 * (b ^ kv4_turn<HD>(p_tok)) + 2 * (lane & 7);
                                *reinterpret_cast<uint16_t *>(stage_p + (kv ? Cfg::VCODES : 0) + r * (HD / 2) + byte) =
                                    (uint16_t)w;
                                if ((lane & 7) == 0) reinterpret_cast<__half *>(kv ? vs : ks)[r * NB + b] = d;
                                if (h0 == 0) {
                                    const int64_t row = row0 + p_tok;
                                    *reinterpret_cast<uint16_t *>((kv ? c.vc : c.kc) + row * (HD / 2) + byte) = (uint16_t)w;
                                    if ((lane & 7) == 0) (kv ? c.vs : c.ks)[row * NB + b] = d;
                                }
                            }
                        }
                        __syncwarp();
                    }
                    // rows that are not seen may hold anything: their scales become zero
                    for (int r = lane; r < TILE; r += 32)
                        if (!seen.sees(p0 + r, a.n_sink)) {
#pragma unroll
                            for (int b = 0; b < NB; b += 2) {
                                *reinterpret_cast<uint32_t *>(ks + (r * NB + b) * 2) = 0u;
                                *reinterpret_cast<uint32_t *>(vs + (r * NB + b) * 2) = 0u;
                            }
                        }
                    // shared memory that a later bulk copy fills again
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }

                // ---- S^T: rows positions 16 hb + gr + {0, 8}, columns heads 2 t4 + {0, 1}
                float s[HB][4];
#pragma unroll
                for (int hb = 0; hb < HB; hb++) {
                    uint32_t w0[NB], w1[NB];  // words t4 of rows gr, gr + 8
                    uint32_t d0[NB / 2], d1[NB / 2];
                    const uint8_t *ks = stage_p + Cfg::KSCALES + (16 * hb + gr) * NB * 2;
                    if constexpr (HD == 128) {
                        ka_ldsm(stage + at_codes + hb * 1024, w0[0], w0[1], w0[2], w0[3]);
                        ka_ldsm(stage + at_codes + hb * 1024 + 512, w1[0], w1[1], w1[2], w1[3]);
                        const uint2 u0 = *reinterpret_cast<const uint2 *>(ks), u1 = *reinterpret_cast<const uint2 *>(ks + 64);
                        d0[0] = u0.x, d0[1] = u0.y, d1[0] = u1.x, d1[1] = u1.y;
                    } else {
                        ka_ldsm(stage + at_codes + hb * 512, w0[0], w0[1], w1[0], w1[1]);
                        d0[0] = *reinterpret_cast<const uint32_t *>(ks), d1[0] = *reinterpret_cast<const uint32_t *>(ks + 32);
                    }
                    s[hb][0] = s[hb][1] = s[hb][2] = s[hb][3] = 0.0f;
                    if constexpr (PREC)
                        ;  // the codes carry their -8
                    else if constexpr (HD == 128)
                        ka_mma8(s[hb], t4 & 1 ? d0[1] : d0[0], t4 & 1 ? d1[1] : d1[0], q_sums);
                    else  // two blocks: lanes t4 = 0 (high) and 2 (low)
                        ka_mma8(s[hb], t4 & 1 ? 0u : d0[0], t4 & 1 ? 0u : d1[0], q_sums);
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            const uint32_t x0 = i ? w0[b] >> 8 : w0[b], x1 = i ? w1[b] >> 8 : w1[b];
                            if constexpr (PREC) {
                                const uint32_t a0 = ka_codes(x0, M1, off1), a1 = ka_codes(x1, M1, off1);
                                const uint32_t a2 = ka_codes(x0, M16, off16), a3 = ka_codes(x1, M16, off16);
                                ka_mma(acc, a0, a1, a2, a3, qh[b][2 * i], qh[b][2 * i + 1]);
                                ka_mma(acc, a0, a1, a2, a3, ql[b][2 * i], ql[b][2 * i + 1]);
                            } else {
                                ka_mma(acc, x0 & M1, x1 & M1, x0 & M16, x1 & M16, qh[b][2 * i], qh[b][2 * i + 1]);
                            }
                        }
                        const float2 f0 = ka_float2(d0[b / 2]), f1 = ka_float2(d1[b / 2]);
                        const float e0 = b & 1 ? f0.y : f0.x, e1 = b & 1 ? f1.y : f1.x;
                        s[hb][0] = fmaf(e0, acc[0], s[hb][0]), s[hb][1] = fmaf(e0, acc[1], s[hb][1]);
                        s[hb][2] = fmaf(e1, acc[2], s[hb][2]), s[hb][3] = fmaf(e1, acc[3], s[hb][3]);
                    }
                }
                if (!whole) {
#pragma unroll
                    for (int hb = 0; hb < HB; hb++)
#pragma unroll
                        for (int i = 0; i < 2; i++)
                            if (!seen.sees(p0 + 16 * hb + gr + 8 * i, a.n_sink)) s[hb][2 * i] = s[hb][2 * i + 1] = -INFINITY;
                }
                // ---- the references and the largest V scale, which seldom grow
                float mx[2];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    mx[i] = fmaxf(s[0][i], s[0][2 + i]);
#pragma unroll
                    for (int hb = 1; hb < HB; hb++) mx[i] = fmaxf(mx[i], fmaxf(s[hb][i], s[hb][2 + i]));
                    mx[i] *= to_log2[i];
                }
                // this lane's share of the V scales, each times its block's factor: the largest
                uint32_t dm = 0;
#pragma unroll
                for (int i = 0; i < Cfg::SCALES; i += 256) {
                    const uint2 u = *reinterpret_cast<const uint2 *>(stage_p + Cfg::VSCALES + i + lane * 8);
                    dm = __vmaxu2(dm, ka_u(__hmul2(ka_h2(u.x & 0x7fff7fffu), ka_h2(room[0]))));
                    dm = __vmaxu2(dm, ka_u(__hmul2(ka_h2(u.y & 0x7fff7fffu), ka_h2(room[NB / 2 - 1]))));
                }
                const bool v_more = (dm + 0x04000400u) & 0xc000c000u;  // 1 (0x3c00) and more
                if (__any_sync(0xffffffffu, mx[0] > ref[0] + KA_ROOM || mx[1] > ref[1] + KA_ROOM || v_more)) {
                    float f[2], fv[NB];
#pragma unroll
                    for (int b = 0; b < NB / 2; b++) {
                        uint32_t d = 0;
#pragma unroll
                        for (int i = 0; i < Cfg::SCALES; i += 256) {
                            const uint2 u = *reinterpret_cast<const uint2 *>(stage_p + Cfg::VSCALES + i + lane * 8);
                            d = __vmaxu2(d, (b ? u.y : u.x) & 0x7fff7fffu);
                            if (NB == 2) d = __vmaxu2(d, u.y & 0x7fff7fffu);
                        }
                        // f16 bits e, m: below 2^(e - 14)
                        const int e0 = (int)(__reduce_max_sync(0xffffffffu, d & 0xffffu) >> 10);
                        const int e1 = (int)(__reduce_max_sync(0xffffffffu, d >> 16) >> 10);
                        const float2 r = ka_float2(room[b]);
                        const float r0 = fminf(r.x, kv4_pow2(14 - e0)), r1 = fminf(r.y, kv4_pow2(14 - e1));
                        room[b] = kv4_half2(r0, r1);
                        fv[2 * b] = r0 * kv4_inv_pow2(r.x), fv[2 * b + 1] = r1 * kv4_inv_pow2(r.y);
                    }
#pragma unroll
                    for (int i = 0; i < 2; i++) {
#pragma unroll
                        for (int m = 4; m <= 16; m <<= 1) mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], m));
                        const float next = fmaxf(ref[i], mx[i]);
                        f[i] = ref[i] == -INFINITY ? 0.0f : kv4_exp2(ref[i] - next);
                        ref[i] = next;
                        l[i] *= f[i];
                    }
#pragma unroll
                    for (int b = 0; b < NB; b++)
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            o[b][i][0] *= f[0] * fv[b], o[b][i][1] *= f[1] * fv[b];
                            o[b][i][2] *= f[0] * fv[b], o[b][i][3] *= f[1] * fv[b];
                        }
                }
                // ---- P (rows positions, columns heads); f32: exact exponents, else 2^KA_BIAS at the reference
                float nr[2];
#pragma unroll
                for (int i = 0; i < 2; i++) nr[i] = (PREC ? 0.0f : KA_BIAS) - (ref[i] == -INFINITY ? 0.0f : ref[i]);
#pragma unroll
                for (int hb = 0; hb < HB; hb++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        s[hb][i] = kv4_exp2(fmaf(s[hb][i], to_log2[i & 1], nr[i & 1]));
                        l[i & 1] += s[hb][i];
                    }
                // ---- O^T += (V^T - 8) (P d): 16 positions a step
                float rf[NB];
#pragma unroll
                for (int b = 0; b < NB; b++) rf[b] = 64.0f * room_of(b);
#pragma unroll
                for (int hb = 0; hb < HB; hb++) {
                    uint32_t ph[NB][2], pl[PREC ? NB : 1][2];  // positions 2 t4 + {0, 1} and + 8, column head gr
                    if constexpr (PREC) {
                        const uint8_t *vs = stage_p + Cfg::VSCALES + (16 * hb + gr) * NB * 2;
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            const float x = s[hb][2 * i], y = s[hb][2 * i + 1];
#pragma unroll
                            for (int b = 0; b < NB; b += 2) {
                                float2 d = ka_float2(*reinterpret_cast<const uint32_t *>(vs + (8 * i * NB + b) * 2));
                                d.x *= rf[b], d.y *= rf[b + 1];
                                uint32_t u, v;
                                ka_split(x * d.x, y * d.x, u, v);
                                ph[b][i] = ka_transpose(u), pl[b][i] = ka_transpose(v);
                                ka_split(x * d.y, y * d.y, u, v);
                                ph[b + 1][i] = ka_transpose(u), pl[b + 1][i] = ka_transpose(v);
                            }
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            const __half2 p = ka_h2(ka_transpose(kv4_half2(s[hb][2 * i], s[hb][2 * i + 1])));
                            const uint8_t *vs = stage_p + Cfg::VSCALES + (16 * hb + 8 * i + 2 * t4) * NB * 2;
                            uint32_t d[NB];  // [position][pair of blocks]
                            if constexpr (HD == 128) {
                                const uint4 u = *reinterpret_cast<const uint4 *>(vs);
                                d[0] = u.x, d[1] = u.y, d[2] = u.z, d[3] = u.w;
                            } else {
                                const uint2 u = *reinterpret_cast<const uint2 *>(vs);
                                d[0] = u.x, d[1] = u.y;
                            }
#pragma unroll
                            for (int b = 0; b < NB; b++) d[b] = ka_u(__hmul2(ka_h2(d[b]), ka_h2(room[b % (NB / 2)])));
#pragma unroll
                            for (int b = 0; b < NB; b++) {
                                const uint32_t dd = __byte_perm(d[b / 2], d[NB / 2 + b / 2], b & 1 ? 0x7632 : 0x5410);
                                ph[b][i] = ka_u(__hmul2(p, ka_h2(dd)));
                            }
                        }
                    }
                    uint32_t x0[NB], x1[NB];  // positions 2 t4 + {0, 1} and + 8, 16-bit unit gr of each block
                    if constexpr (HD == 128) {
                        ka_ldsm_t(stage + Cfg::VCODES + at_codes + hb * 1024, x0[0], x0[1], x0[2], x0[3]);
                        ka_ldsm_t(stage + Cfg::VCODES + at_codes + hb * 1024 + 512, x1[0], x1[1], x1[2], x1[3]);
                    } else {
                        ka_ldsm_t(stage + Cfg::VCODES + at_codes + hb * 512, x0[0], x0[1], x1[0], x1[1]);
                    }
#pragma unroll
                    for (int b = 0; b < NB; b++)
#pragma unroll
                        for (int i = 0; i < 2; i++) {  // rows: values 4 gr + 2 i, and 4 gr + 2 i + 1 (16 times)
                            const uint32_t y0 = i ? x0[b] >> 8 : x0[b], y1 = i ? x1[b] >> 8 : x1[b];
                            const uint32_t a0 = ka_codes(y0, M1, off1), a1 = ka_codes(y0, M16, off16);
                            const uint32_t a2 = ka_codes(y1, M1, off1), a3 = ka_codes(y1, M16, off16);
                            ka_mma(o[b][i], a0, a1, a2, a3, ph[b][0], ph[b][1]);
                            if constexpr (PREC) ka_mma(o[b][i], a0, a1, a2, a3, pl[b][0], pl[b][1]);
                        }
                }
            }
            __syncwarp();  // every lane is done with the stage
            if (!dead && filled < mine) {
                fill(filled);
                filled++;
            }
        }

        if (__builtin_expect(!held && !dead && __any_sync(0xffffffffu, kv4_far(ref[0]) || kv4_far(ref[1])), 0)) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int far = kv4_far(ref[i]);
                to_log2[i] *= kv4_pow2(-far);
                if (gr == 0) sh_up[warp][2 * t4 + i] = kv4_pow2(far);
            }
            held = true;
            fill_first();
            goto tiles;
        }

        // ---- join the warps: [warp][head][ref, l, o...]
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int m = 4; m <= 16; m <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], m);
        __syncthreads();  // the ring is idle
        float *sums = reinterpret_cast<float *>(ka_smem);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            float *r = sums + (warp * KA_HEADS + 2 * t4 + i) * RW;
            if (gr == 0) r[0] = held ? ref[i] * sh_up[warp][2 * t4 + i] : ref[i], r[1] = l[i];
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const float f = (PREC ? 0.015625f : 1.0f) * kv4_inv_pow2(room_of(b));
#pragma unroll
                for (int e = 0; e < 2; e++)
                    *reinterpret_cast<float2 *>(r + 2 + 32 * b + 4 * gr + 2 * e) =
                        make_float2(o[b][e][i] * f, o[b][e][2 + i] * (f * 0.0625f));
            }
        }
        __syncthreads();
        const bool split = parts > 1;
        // A run's part of a segment that started in an earlier run is in its slot 0, else in slot 1
        float *mine_out = a.part + ((int64_t)run * 2 + (run == first_run)) * KA_HEADS * RW;
        T *out = reinterpret_cast<T *>(a.out) + (int64_t)t * a.out_ld + (int64_t)(g * G + h0) * HD;
        // A thread joins 4 values of a head at a time.  A sum whose reference is still -inf counts only if it is not
        // zero (a NaN, which must come out)
        struct Sum {
            float top = -INFINITY, l = 0.0f, x[4] = {0, 0, 0, 0};
            __device__ __forceinline__ void add(float r, float l_, float2 y0, float2 y1) {
                if (l_ == 0.0f) return;
                const float f = r == -INFINITY ? 1.0f : kv4_exp2(r - top);
                l += f * l_;
                x[0] += f * y0.x, x[1] += f * y0.y, x[2] += f * y1.x, x[3] += f * y1.y;
            }
            __device__ __forceinline__ void store(T *p) const {
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                if constexpr (sizeof(T) == 4)
                    *reinterpret_cast<float4 *>(p) = make_float4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
                else
                    *reinterpret_cast<uint2 *>(p) =
                        make_uint2(kv4_pack_bf2(x[0] * inv, x[1] * inv), kv4_pack_bf2(x[2] * inv, x[3] * inv));
            }
        };
#pragma unroll 1
        for (int i = threadIdx.x; i < heads * (HD / 4); i += Cfg::THREADS) {
            const int h = i / (HD / 4), d = 4 * (i % (HD / 4));
            Sum sum;
#pragma unroll
            for (int w = 0; w < WARPS; w++) sum.top = fmaxf(sum.top, sums[(w * KA_HEADS + h) * RW]);
#pragma unroll
            for (int w = 0; w < WARPS; w++) {
                const float *r = sums + (w * KA_HEADS + h) * RW;
                sum.add(r[0], r[1], *reinterpret_cast<const float2 *>(r + 2 + d), *reinterpret_cast<const float2 *>(r + 4 + d));
            }
            if (split) {
                float2 *r = reinterpret_cast<float2 *>(mine_out + h * RW);
                if (d == 0) r[0] = make_float2(sum.top, sum.l);
                r[1 + d / 2] = make_float2(sum.x[0], sum.x[1]), r[2 + d / 2] = make_float2(sum.x[2], sum.x[3]);
            } else {
                sum.store(out + h * HD + d);
            }
        }
        if (split) {
            __syncthreads();
            if (threadIdx.x == 0) {
                int n;  // release this CTA's part, acquire the others'
                asm volatile("fence.acq_rel.gpu; atom.add.acq_rel.gpu.s32 %0, [%1], 1;" : "=r"(n) : "l"(a.arrived + first_run) : "memory");
                sh_last = n == parts - 1;
                if (sh_last) a.arrived[first_run] = 0;
            }
            __syncthreads();
#pragma unroll 1
            for (int i = threadIdx.x; sh_last && i < heads * (HD / 4); i += Cfg::THREADS) {
                const int h = i / (HD / 4), d = 4 * (i % (HD / 4));
                const float *p = a.part + ((int64_t)first_run * 2 * KA_HEADS + h) * RW;
                Sum sum;
#pragma unroll 1
                for (int w0 = 0; w0 < parts; w0 += 8) {
                    float2 rl[8], y0[8], y1[8];
#pragma unroll
                    for (int w = 0; w < 8; w++) {
                        rl[w] = make_float2(-INFINITY, 0.0f), y0[w] = y1[w] = make_float2(0.0f, 0.0f);
                        if (w0 + w < parts) {
                            const float2 *r = reinterpret_cast<const float2 *>(p + ((w0 + w) * 2 + (w0 + w == 0)) * (KA_HEADS * RW));
                            rl[w] = __ldcg(r), y0[w] = __ldcg(r + 1 + d / 2), y1[w] = __ldcg(r + 2 + d / 2);
                        }
                    }
                    float top = sum.top;
#pragma unroll
                    for (int w = 0; w < 8; w++) top = fmaxf(top, rl[w].x);
                    const float f = sum.top == -INFINITY ? 1.0f : kv4_exp2(sum.top - top);
                    sum.l *= f, sum.x[0] *= f, sum.x[1] *= f, sum.x[2] *= f, sum.x[3] *= f;
                    sum.top = top;
#pragma unroll
                    for (int w = 0; w < 8; w++) sum.add(rl[w].x, rl[w].y, y0[w], y1[w]);
                }
                sum.store(out + h * HD + d);
            }
        }
        __syncthreads();  // the sums are read; the ring may be filled again
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
}

// ------------------------------------------------------------------ launchers
template <int HD, typename T>
static cudaError_t rows_launch(bool store, void *k, void *v, int64_t ld, const int32_t *seq, int seq0,
                               const int32_t *pos, int pos0, int64_t n, const Kv4Planes &c, int *err, cudaStream_t st) {
    const dim3 grid((unsigned)((n * (HD / (store ? 16 : 8)) + 255) / 256), 2 * c.n_kv);
    const Kv4RowArgs a{k, v, ld, n, seq, pos, seq0, pos0, c, err};
    return launch_k(store ? kv4_store_kernel<HD, T> : kv4_load_kernel<HD, T>, grid, dim3(256), 0, st, a);
}

cudaError_t launch_kv4_rows(bool store, bool f32, int head_dim, void *k, void *v, int64_t ld, const int32_t *seq,
                            int seq0, const int32_t *pos, int pos0, int64_t n, const Kv4Planes &c, int *err,
                            cudaStream_t st) {
    if (n <= 0) return cudaSuccess;
    if (n > (1ll << 30) || c.n_kv > 32767) return cudaErrorInvalidValue;
    if (head_dim == 128)
        return f32 ? rows_launch<128, float>(store, k, v, ld, seq, seq0, pos, pos0, n, c, err, st)
                   : rows_launch<128, __nv_bfloat16>(store, k, v, ld, seq, seq0, pos, pos0, n, c, err, st);
    return f32 ? rows_launch<64, float>(store, k, v, ld, seq, seq0, pos, pos0, n, c, err, st)
               : rows_launch<64, __nv_bfloat16>(store, k, v, ld, seq, seq0, pos, pos0, n, c, err, st);
}

size_t kv4_attn_scratch_bytes(int sm_count) {
    const size_t runs = 2 * (size_t)sm_count, decode = runs * 2 * KA_HEADS * (128 + 2) * 4;
    const size_t prefill = kv4_prefill_part_bytes(sm_count);
    return kv4_counter_bytes(sm_count) + (decode > prefill ? decode : prefill);
}

template <int HD, typename T, bool SHORT>
static cudaError_t attn_launch(const Kv4Attn &x, const Kv4Planes &c, int64_t segments, int64_t tiles, void *scratch, int sm_count,
                               int *err, cudaStream_t st) {
    using Cfg = Kv4AttnCfg<HD, sizeof(T) == 4, SHORT>;
    static int set[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!set[dev]) {
        const cudaError_t e =
            cudaFuncSetAttribute(kv4_attn_kernel<HD, T, SHORT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM);
        if (e != cudaSuccess) return e;
        set[dev] = 1;
    }
    // as many CTAs as the most tiles that the cache allows need, at a tile a warp, and at most what is resident
    const int64_t want = segments + (tiles + Cfg::WARPS - 1) / Cfg::WARPS, cap = (int64_t)Cfg::CTAS * sm_count;
    Kv4AttnArgs a;
    a.q = x.q, a.k = x.k, a.v = x.v, a.out = x.out;
    a.q_ld = x.q_ld, a.kv_ld = x.kv_ld, a.out_ld = x.out_ld;
    a.pos = x.pos, a.pos0 = x.pos0, a.seq0 = x.seq0;
    a.n_tok = x.n_tok, a.n_head = x.n_head, a.window = x.window, a.n_sink = x.n_sink, a.scale = x.scale;
    a.arrived = (int *)scratch;
    a.part = kv4_scratch_parts(scratch, sm_count);
    a.err = err;
    return launch_k(kv4_attn_kernel<HD, T, SHORT>, dim3((unsigned)(want < cap ? want : cap)), dim3(Cfg::THREADS),
                    (size_t)Cfg::SMEM, st, a, c);
}

cudaError_t launch_kv4_attn(bool f32, int head_dim, Kv4Attn &x, const Kv4Planes &c, void *scratch, int sm_count,
                            int *err, cudaStream_t st) {
    if (x.n_tok <= 0) return cudaSuccess;
    // The most tiles that a token can see, as far as the host knows: decode positions are on the device, so that without a window
    // it is the cache's capacity.  Sequences well below it then take the other form: 128 of 2048 positions 48 us in a cache of
    // 2048, 58 in one of 32768; 64 of 4096 44 and 48.
    constexpr int TILE = 64;
    const int G = x.n_head / c.n_kv, passes = (G + KA_HEADS - 1) / KA_HEADS;
    int64_t most = x.pos ? c.n_ctx : x.pos0 + x.n_tok;
    if (x.window > 0) most = std::min(most, (int64_t)x.window + 2 * TILE + x.n_sink);
    const int64_t each = (std::min(most, (int64_t)c.n_ctx) + TILE - 1) / TILE;
    const int64_t segments = (int64_t)x.n_tok * c.n_kv * passes, tiles = segments * each;
    if (tiles + 32 * segments > (1ll << 30)) return cudaErrorInvalidValue;  // list positions are 32-bit
    const bool few_tiles = segments > sm_count && each <= 128;
    auto launch = [&](auto kernel) { return kernel(x, c, segments, tiles, scratch, sm_count, err, st); };
    if (head_dim == 64) return launch(f32 ? attn_launch<64, float, false> : attn_launch<64, __nv_bfloat16, false>);
    if (few_tiles) return launch(f32 ? attn_launch<128, float, true> : attn_launch<128, __nv_bfloat16, true>);
    return launch(f32 ? attn_launch<128, float, false> : attn_launch<128, __nv_bfloat16, false>);
}

}  // namespace tmoe
