// The 4-bit KV cache (format: kv4.cuh): quantising rows into it, reading rows back, and the attention
// of single query tokens over it.
//   kv4_store_kernel   K and V rows -> codes and scales, at any (sequence, position) of each row
//   kv4_load_kernel    the same rows back as values
//   kv4_attn_kernel    one query token per sequence (a decode step), its K/V row quantised into the
//                      cache on the way; or a few tokens of one sequence
#include "kernels.cuh"
#include "kv4.cuh"

namespace tmoe {

// ------------------------------------------------------------------ rows in and out
// Row i of a call: its sequence and position; false: no row.  A negative position means "no row" to
// the caller too; any other place outside the cache latches the device error.
__device__ __forceinline__ bool kv4_place(const int32_t *seq, int seq0, const int32_t *pos, int pos0, int64_t i,
                                          const Kv4Planes &c, int *err, int &s, int &p) {
    const int64_t ps = pos ? pos[i] : pos0 + i, sq = seq ? seq[i] : seq0 >= 0 ? seq0 : i;
    if (ps < 0) return false;
    if (ps >= c.n_ctx || sq < 0 || sq >= c.n_seq) {
        latch_error(err, TMOE_DEV_ERR_BADPOS);
        return false;
    }
    s = (int)sq, p = (int)ps;
    return true;
}

// Rows are independent and only moved once: HBM-bound.  A thread takes 8 values (a block is 4 threads,
// its extremes two shuffles each way), so that a warp reads whole 128-byte lines and writes 8 blocks'
// chunks; rows run fastest over the threads, so that a run of positions writes one contiguous piece of a
// head's plane.
template <int HD, typename T>
__global__ void __launch_bounds__(256) kv4_store_kernel(const T *__restrict__ k, const T *__restrict__ v, int64_t ld,
                                                        const int32_t *__restrict__ seq, int seq0,
                                                        const int32_t *__restrict__ pos, int pos0, int64_t n,
                                                        Kv4Planes c, int *err) {
    constexpr int TPR = HD / 8, NB = HD / 32;
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t i = at / TPR;
    const int sub = (int)(at % TPR), b = sub >> 2;
    const int g = blockIdx.y >> 1;
    const bool is_v = blockIdx.y & 1;
    pdl_wait();
    pdl_trigger();
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    int s = 0, p = 0;
    const bool ok = i < n && kv4_place(seq, seq0, pos, pos0, i, c, err, s, p);
    if (ok) kv4_load_row((is_v ? v : k) + i * ld + (int64_t)g * HD + 8 * sub, x);
    float hi = -FLT_MAX, lo = FLT_MAX;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        x[j] = kv4_finite(x[j]);
        hi = fmaxf(hi, x[j]), lo = fminf(lo, x[j]);
    }
#pragma unroll
    for (int o = 1; o <= 2; o <<= 1) {
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    }
    __half d;
    float inv;
    kv4_scale(hi, lo, d, inv);
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) w |= kv4_code(x[j], inv) << (4 * j);
    if (!ok) return;
    const int64_t row = ((int64_t)s * c.n_kv + g) * c.n_ctx + p;
    uint8_t *codes = (is_v ? c.vc : c.kc) + row * (HD / 2);
    *reinterpret_cast<uint32_t *>(codes + 16 * (b ^ kv4_turn<HD>(p)) + 4 * (sub & 3)) = w;
    if ((sub & 3) == 0) (is_v ? c.vs : c.ks)[row * NB + b] = d;
}

template <int HD, typename T>
__global__ void __launch_bounds__(256) kv4_load_kernel(T *__restrict__ k, T *__restrict__ v, int64_t ld,
                                                       const int32_t *__restrict__ seq, int seq0,
                                                       const int32_t *__restrict__ pos, int pos0, int64_t n,
                                                       Kv4Planes c, int *err) {
    constexpr int TPR = HD / 8, NB = HD / 32;
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t i = at / TPR;
    const int sub = (int)(at % TPR), b = sub >> 2;
    const int g = blockIdx.y >> 1;
    const bool is_v = blockIdx.y & 1;
    pdl_wait();
    pdl_trigger();
    if (i >= n) return;
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    int s, p;
    if (kv4_place(seq, seq0, pos, pos0, i, c, err, s, p)) {
        const int64_t row = ((int64_t)s * c.n_kv + g) * c.n_ctx + p;
        const uint8_t *codes = (is_v ? c.vc : c.kc) + row * (HD / 2);
        const uint32_t w = *reinterpret_cast<const uint32_t *>(codes + 16 * (b ^ kv4_turn<HD>(p)) + 4 * (sub & 3));
        const float d = __half2float((is_v ? c.vs : c.ks)[row * NB + b]);
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = d * (float)((int)((w >> (4 * j)) & 15u) - 8);
    }
    kv4_store_row((is_v ? v : k) + i * ld + (int64_t)g * HD + 8 * sub, x);
}

// ------------------------------------------------------------------ attention of single tokens
// For each query token and KV head: softmax(q K^T) V over the seen positions, up to 8 of the head's query
// heads together (more are further passes over the same rows, from L2).
//
// Bound: HBM (a cached position is read once, 4.5 bits a value).  At that rate an SM has about 195
// clocks for a 32-position tile of 128-wide K and V, 780 issue slots; the kernel needs about 500 of
// them (f32 queries: 620), so the work per value has to stay small:
//   - Codes meet the tensor cores as they are.  S = Q K^T runs on mma.sync m16n8k16 (f16 operands, f32
//     sums) with the heads as rows: a 4-bit code under a mask is the f16 subnormal c * 2^-24 (or 16 times
//     that), so a word of 8 codes becomes four operand registers with four ANDs and one shift.  The
//     factor 16 is undone in Q, the -8 is the accumulator's start value -8 * sum(q), and the scale of
//     a block multiplies its own accumulator in f32: K enters exactly.
//   - O += P V takes V the same way, as 1024 + c minus 1032 in f16 (here the -8 has to go before the
//     product: averaged over many positions, sum(P c) - 8 sum(P) would cancel), its scale on P.
//   - No transposes: K's words through ldmatrix are the B operand for two steps of 16 dimensions; V's 16-bit
//     units (4 codes) through ldmatrix.trans are, mask by mask, the B operand of four output blocks,
//     and S's accumulators are P's A operand.
// Precision: Q is scaled by a power of two per head into f16's upper range; bf16 queries then are exact.
// f32 queries are split as high + low f16 parts, the low ones in rows 8..15 of the operand, which the
// 8 heads leave free; P likewise.  P times the V scale is held relative to the running maximum and the
// largest V scale seen, so that small scales do not end in f16's subnormals; for bf16 it is one f16
// (2^-12 relative, below the output's own 2^-9).
//
// Work: the tiles of all (token, KV head, pass) are one list, cut into equal runs, one per CTA: ragged
// lengths, few sequences or many all load every SM the same.  A warp takes every 8th tile of a run,
// fetched by bulk copies into its own ring.  Runs that end inside a token's list leave partial sums in
// scratch; the CTA that arrives last there joins them, in run order (same sums every call).
constexpr int KA_TILE = 32;
constexpr int KA_WARPS = 8;
constexpr int KA_THREADS = 32 * KA_WARPS;
constexpr int KA_HEADS = 8;

struct Kv4AttnArgs {
    const void *q, *k, *v;  // k == nullptr: the new rows are in the cache already
    void *out;
    int64_t q_ld, kv_ld, out_ld;
    const int32_t *pos;  // nullptr: token t at pos0 + t
    int pos0, seq0;      // seq0 >= 0: every token is of that sequence; else token t of sequence t
    int n_tok, n_head, window, n_sink;
    float scale;
    int *arrived;  // [grid] zero between calls
    float *part;   // [2 * grid][KA_HEADS][HD + 2]
    int *err;
};

template <int HD, bool PREC>
struct Kv4AttnCfg {
    static constexpr int NB = HD / 32;
    static constexpr int CODES = KA_TILE * HD / 2, SCALES = KA_TILE * NB * 2;
    static constexpr int STAGE = 2 * (CODES + SCALES);
    static constexpr int STAGES = (PREC ? 6 : 3) * (128 / HD);
    static constexpr int CTAS = PREC ? 1 : 2;  // per SM
    static constexpr int RING = KA_WARPS * STAGES * STAGE;
    static constexpr int SMEM = RING + KA_WARPS * STAGES * 8 + 128;
    static_assert(KA_WARPS * KA_HEADS * (HD + 2) * 4 <= RING, "the warps' sums are joined in the ring's space");
};

__device__ __forceinline__ void ka_ldsm(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ void ka_ldsm_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
// d = a b + c; without PREC rows 8..15 of a are zero and their results are dropped.
template <bool PREC>
__device__ __forceinline__ void ka_mma(float (&d)[PREC ? 4 : 2], const float (&c)[PREC ? 4 : 2], uint32_t a0, uint32_t a1,
                                       uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (PREC) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
    } else {
        float x, y;
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(x), "=f"(y)
            : "r"(a0), "r"(0u), "r"(a2), "r"(0u), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(0.0f), "f"(0.0f));
    }
}
__device__ __forceinline__ float2 ka_float2(uint32_t u) {
    __half2 h;
    memcpy(&h, &u, 4);
    return __half22float2(h);
}
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
    __half2 h;
    memcpy(&h, &r, 4);
    h = __hsub2(h, off);
    memcpy(&r, &h, 4);
    return r;
}

template <int HD, typename T>
__global__ void __launch_bounds__(KA_THREADS, (Kv4AttnCfg<HD, sizeof(T) == 4>::CTAS))
    kv4_attn_kernel(const Kv4AttnArgs a, const Kv4Planes c) {
    constexpr bool PREC = sizeof(T) == 4;
    using Cfg = Kv4AttnCfg<HD, PREC>;
    constexpr int NB = Cfg::NB, AC = PREC ? 4 : 2, ST = Cfg::STAGES;
    extern __shared__ __align__(128) uint8_t ka_smem[];
    uint64_t *bars = reinterpret_cast<uint64_t *>(ka_smem + Cfg::RING);
    __shared__ long long sh_sum[KA_WARPS];
    __shared__ long long sh_start[2];  // token and the list position of its first tile
    __shared__ int sh_last;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gr = lane >> 2, t4 = lane & 3;
    const int G = a.n_head / c.n_kv, passes = (G + KA_HEADS - 1) / KA_HEADS, H = c.n_kv * passes;
    uint8_t *ring = ka_smem + warp * ST * Cfg::STAGE;
    uint64_t *bar = bars + warp * ST;
    if (lane == 0)
        for (int s = 0; s < ST; s++) mbar_init(&bar[s], 1);
    fence_barrier_init();
    pdl_wait();
    pdl_trigger();

    auto pos_of = [&](int t) -> int {  // -1: no query
        const int64_t p = a.pos ? a.pos[t] : (int64_t)a.pos0 + t;
        if (p >= c.n_ctx) return -2;
        return p < 0 ? -1 : (int)p;
    };
    auto tiles_of = [&](int t) -> int {
        if (t >= a.n_tok) return 0;
        const int p = pos_of(t);
        return p < 0 ? 0 : Kv4Seen::of<KA_TILE>(p, a.window, a.n_sink).tiles;
    };
    // the list: token t's tiles, H times (once per KV head and pass), t ascending.  Its length, and
    // where this CTA's run starts
    auto scan = [&](int base, long long &before, long long &sum) -> int {  // over 256 tokens; a CTA barrier inside
        const int n = tiles_of(base + threadIdx.x);
        long long inc = n;
        for (int o = 1; o < 32; o <<= 1) {
            const long long up = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += up;
        }
        if (lane == 31) sh_sum[warp] = inc;
        __syncthreads();
        before = inc - n, sum = 0;
        for (int w = 0; w < KA_WARPS; w++) {
            if (w < warp) before += sh_sum[w];
            sum += sh_sum[w];
        }
        __syncthreads();
        return n;
    };
    long long total = 0, before = 0, sum = 0;
    int n_mine = 0;
    for (int base = 0; base < a.n_tok; base += KA_THREADS) {
        n_mine = scan(base, before, sum);
        total += sum;
    }
    total *= H;
    const long long even = (total + gridDim.x - 1) / gridDim.x;
    const long long per = even > KA_WARPS ? even : KA_WARPS;  // a tile for each warp before another CTA joins in
    const long long start = blockIdx.x * per, end = start + per < total ? start + per : total;
    // tokens without a query: zeros
    for (int t = blockIdx.x; t < a.n_tok; t += gridDim.x) {
        const int p = pos_of(t);
        if (p >= 0) continue;
        if (p == -2 && threadIdx.x == 0) latch_error(a.err, TMOE_DEV_ERR_BADPOS);
        T *o = reinterpret_cast<T *>(a.out) + (int64_t)t * a.out_ld;
        const float z[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        for (int i = threadIdx.x; i < a.n_head * HD / 8; i += KA_THREADS) kv4_store_row(o + 8 * i, z);
    }
    if (start >= end) return;
    long long run = 0;
    for (int base = 0; base < a.n_tok; base += KA_THREADS) {
        if (a.n_tok > KA_THREADS) n_mine = scan(base, before, sum);
        const long long s0 = (run + before) * H;
        if (n_mine && s0 <= start && start < s0 + (long long)n_mine * H) sh_start[0] = base + threadIdx.x, sh_start[1] = s0;
        run += sum;
    }
    __syncthreads();
    int tok = (int)sh_start[0];
    long long tok0 = sh_start[1];  // list position of the token's first tile
    long long at = start;
    int fills = 0;  // of this warp's ring, over all parts of the run

    while (at < end) {
        const int p_new = pos_of(tok);
        if (p_new < 0) {
            tok++;
            continue;
        }
        const Kv4Seen seen = Kv4Seen::of<KA_TILE>(p_new, a.window, a.n_sink);
        const int hc = (int)((at - tok0) / seen.tiles), first = (int)((at - tok0) % seen.tiles);
        const long long seg0 = tok0 + (long long)hc * seen.tiles;  // the list position of this head's tiles
        const int n_part = (int)(end - at < seen.tiles - first ? end - at : seen.tiles - first);
        const int g = hc / passes, h0 = (hc % passes) * KA_HEADS;
        const int heads = G - h0 < KA_HEADS ? G - h0 : KA_HEADS;
        const int sq = a.seq0 >= 0 ? a.seq0 : tok;
        const int64_t row0 = ((int64_t)sq * c.n_kv + g) * c.n_ctx;

        // ---- this warp's tiles: first + warp, first + warp + 8, ...
        const int mine = n_part > warp ? (n_part - warp + KA_WARPS - 1) / KA_WARPS : 0;
        auto fill = [&](int j) {
            if (lane == 0) {
                const int s = (fills + j) % ST;
                const int64_t r = row0 + (int64_t)seen.tile(first + warp + j * KA_WARPS) * KA_TILE;
                uint8_t *d = ring + s * Cfg::STAGE;
                mbar_arrive_expect_tx(&bar[s], Cfg::STAGE);
                bulk_g2s(d, c.kc + r * (HD / 2), Cfg::CODES, &bar[s]);
                bulk_g2s(d + Cfg::CODES, c.ks + r * NB, Cfg::SCALES, &bar[s]);
                bulk_g2s(d + Cfg::CODES + Cfg::SCALES, c.vc + r * (HD / 2), Cfg::CODES, &bar[s]);
                bulk_g2s(d + 2 * Cfg::CODES + Cfg::SCALES, c.vs + r * NB, Cfg::SCALES, &bar[s]);
            }
        };
        int filled = 0;
        for (; filled < mine && filled < ST; filled++) fill(filled);

        // ---- Q operand: head gr of the pass; of block b the thread has dims 32 b + 8 t4 + 0..7, as
        // pairs (0, 4), (1, 5) / 16, (2, 6), (3, 7) / 16, matching the codes' order in a word
        uint32_t qh[NB][4], ql[PREC ? NB : 1][4];
        float start_acc[NB][AC];
        float to_log2;
        {
            float x[NB][8];
            float top = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; b++) {
#pragma unroll
                for (int i = 0; i < 8; i++) x[b][i] = 0.0f;
                if (gr < heads)
                    kv4_load_row(reinterpret_cast<const T *>(a.q) + (int64_t)tok * a.q_ld +
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
            to_log2 = a.scale * 1.4426950408889634f * kv4_pow2(12 - e1) * kv4_pow2(12 - e2);
#pragma unroll
            for (int b = 0; b < NB; b++) {
                float z[8], sh = 0.0f, sl = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) z[i] = x[b][i] * up1 * up2;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float2 f;
                    if constexpr (PREC) {
                        ka_split(z[i], z[i + 4], qh[b][i], ql[b][i]);
                        f = ka_float2(ql[b][i]);
                        sl += f.x + f.y;
                    } else {
                        qh[b][i] = kv4_half2(z[i], z[i + 4]);
                    }
                    f = ka_float2(qh[b][i]);
                    sh += f.x + f.y;
                    if (i & 1) {
                        const __half2 r = __float2half2_rn(0.0625f);
                        __half2 h;
                        memcpy(&h, &qh[b][i], 4);
                        h = __hmul2(h, r);
                        memcpy(&qh[b][i], &h, 4);
                        if constexpr (PREC) {
                            memcpy(&h, &ql[b][i], 4);
                            h = __hmul2(h, r);
                            memcpy(&ql[b][i], &h, 4);
                        }
                    }
                }
                sh += __shfl_xor_sync(0xffffffffu, sh, 1);
                sh += __shfl_xor_sync(0xffffffffu, sh, 2);
                start_acc[b][0] = start_acc[b][1] = -8.0f * 0x1p-24f * sh;
                if constexpr (PREC) {
                    sl += __shfl_xor_sync(0xffffffffu, sl, 1);
                    sl += __shfl_xor_sync(0xffffffffu, sl, 2);
                    start_acc[b][2] = start_acc[b][3] = -8.0f * 0x1p-24f * sl;
                }
            }
        }
        float o[NB][4][AC];
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < AC; j++) o[b][i][j] = 0.0f;
        // of head gr: the running maximum; what exponents are taken against (the maximum, lowered by the
        // room that P times the largest V scale leaves below 2^14); the sum, over this thread's positions
        float top = -INFINITY, ref = -INFINITY, l = 0.0f;
        uint32_t v_top = 0;     // the largest V scale seen, as f16 bits
        int v_exp = 0;          // V scales are below 2^v_exp
        const __half2 off1 = __float2half2_rn(1032.0f), off16 = __float2half2_rn(1152.0f);
        bool dead = false;

        for (int j = 0; j < filled; j++) {
            const int s = (fills + j) % ST;
            if (!__all_sync(0xffffffffu, mbar_wait_bounded(&bar[s], ((fills + j) / ST) & 1))) {
                if (lane == 0) latch_error(a.err, TMOE_DEV_ERR_TIMEOUT);
                dead = true;  // no more fills; the loop goes on to wait for those in flight
            }
            uint8_t *kcodes = ring + s * Cfg::STAGE, *kscales = kcodes + Cfg::CODES, *vcodes = kscales + Cfg::SCALES,
                    *vscales = vcodes + Cfg::CODES;
            const int tile = seen.tile(first + warp + j * KA_WARPS), p0 = tile * KA_TILE;
            const bool whole = seen.whole(p0, KA_TILE, a.n_sink);
            if (!dead) {
                if (a.k && tile == p_new / KA_TILE) {
                    // the new row: quantised into the tile, and (one pass only) into the cache
                    constexpr int LANES = HD / 4;
                    const int r = p_new % KA_TILE, b = lane >> 3;
#pragma unroll
                    for (int kv = 0; kv < 2; kv++) {
                        float x[4] = {0, 0, 0, 0};
                        if (lane < LANES)
                            kv4_load_row(reinterpret_cast<const T *>(kv ? a.v : a.k) + (int64_t)tok * a.kv_ld + g * HD +
                                             4 * lane, x);
                        float hi = -FLT_MAX, lo = FLT_MAX;
#pragma unroll
                        for (int i = 0; i < 4; i++) x[i] = kv4_finite(x[i]), hi = fmaxf(hi, x[i]), lo = fminf(lo, x[i]);
#pragma unroll
                        for (int m = 1; m <= 4; m <<= 1) {
                            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, m));
                            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, m));
                        }
                        __half d;
                        float inv;
                        kv4_scale(hi, lo, d, inv);
                        uint32_t w = 0;
#pragma unroll
                        for (int i = 0; i < 4; i++) w |= kv4_code(x[i], inv) << (4 * i);
                        if (lane < LANES) {
                            const int byte = 16 * (b ^ kv4_turn<HD>(p_new)) + 2 * (lane & 7);
                            uint8_t *sc = kv ? vcodes : kcodes;
                            __half *ss = reinterpret_cast<__half *>(kv ? vscales : kscales);
                            *reinterpret_cast<uint16_t *>(sc + r * (HD / 2) + byte) = (uint16_t)w;
                            if ((lane & 7) == 0) ss[r * NB + b] = d;
                            if (h0 == 0) {
                                const int64_t row = row0 + p_new;
                                *reinterpret_cast<uint16_t *>((kv ? c.vc : c.kc) + row * (HD / 2) + byte) = (uint16_t)w;
                                if ((lane & 7) == 0) (kv ? c.vs : c.ks)[row * NB + b] = d;
                            }
                        }
                    }
                    __syncwarp();
                }
                if (!whole && !seen.sees(p0 + lane, a.n_sink)) {
                    // rows that are not seen may hold anything: their scales become zero
#pragma unroll
                    for (int b = 0; b < NB; b += 2) {
                        *reinterpret_cast<uint32_t *>(kscales + (lane * NB + b) * 2) = 0u;
                        *reinterpret_cast<uint32_t *>(vscales + (lane * NB + b) * 2) = 0u;
                    }
                }
                // both wrote shared memory that a later bulk copy fills again
                if (!whole || tile == p_new / KA_TILE) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();

                // ---- S: 8 heads x 32 positions; this thread: head gr, positions 8 nb + 2 t4 + {0, 1}
                float sc[4][2];
                const uint32_t k_at = smem_u32(kcodes), v_at = smem_u32(vcodes);
#pragma unroll
                for (int nb = 0; nb < 4; nb++) {
                    uint32_t w[4];
                    uint32_t ds[NB];  // scales of the two positions, [position][block]
                    if constexpr (HD == 128) {
                        const int r = 8 * nb + (lane & 7), b = lane >> 3;
                        ka_ldsm(k_at + r * 64 + 16 * (b ^ kv4_turn<128>(r)), w);
                        const uint4 d4 = *reinterpret_cast<const uint4 *>(kscales + (8 * nb + 2 * t4) * 8);
                        ds[0] = d4.x, ds[1] = d4.y, ds[2] = d4.z, ds[3] = d4.w;
                    } else {
                        const int r = 8 * nb + (lane & 7), b = (lane >> 3) & 1;  // lanes 16..31: the same again
                        ka_ldsm(k_at + r * 32 + 16 * (b ^ kv4_turn<64>(r)), w);
                        const uint2 d2 = *reinterpret_cast<const uint2 *>(kscales + (8 * nb + 2 * t4) * 4);
                        ds[0] = d2.x, ds[1] = d2.y;
                    }
                    float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        float acc[AC], acc2[AC];
                        const uint32_t w8 = w[b] >> 8;
                        constexpr uint32_t M1 = 0x000f000fu, M16 = 0x00f000f0u;
                        ka_mma<PREC>(acc, start_acc[b], qh[b][0], PREC ? ql[PREC ? b : 0][0] : 0, qh[b][1],
                                     PREC ? ql[PREC ? b : 0][1] : 0, w[b] & M1, w[b] & M16);
                        ka_mma<PREC>(acc2, acc, qh[b][2], PREC ? ql[PREC ? b : 0][2] : 0, qh[b][3],
                                     PREC ? ql[PREC ? b : 0][3] : 0, w8 & M1, w8 & M16);
                        if constexpr (PREC) acc2[0] += acc2[AC - 2], acc2[1] += acc2[AC - 1];
                        const float2 d0 = ka_float2(ds[b / 2]), d1 = ka_float2(ds[NB / 2 + b / 2]);
                        s0 = fmaf(b & 1 ? d0.y : d0.x, acc2[0], s0);
                        s1 = fmaf(b & 1 ? d1.y : d1.x, acc2[1], s1);
                    }
                    sc[nb][0] = s0 * to_log2, sc[nb][1] = s1 * to_log2;
                }
                if (!whole) {
#pragma unroll
                    for (int nb = 0; nb < 4; nb++)
#pragma unroll
                        for (int i = 0; i < 2; i++)
                            if (!seen.sees(p0 + 8 * nb + 2 * t4 + i, a.n_sink)) sc[nb][i] = -INFINITY;
                }
                // ---- the running maximum and the largest V scale; both seldom grow
                float mx = sc[0][0];
#pragma unroll
                for (int nb = 0; nb < 4; nb++) mx = fmaxf(mx, fmaxf(sc[nb][0], sc[nb][1]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                uint32_t dm;  // this lane's position: its largest V scale
                if constexpr (HD == 128) {
                    const uint2 u = *reinterpret_cast<const uint2 *>(vscales + lane * 8);
                    dm = __vmaxu2(u.x & 0x7fff7fffu, u.y & 0x7fff7fffu);
                } else {
                    dm = *reinterpret_cast<const uint32_t *>(vscales + lane * 4) & 0x7fff7fffu;
                }
                dm = max(dm & 0xffffu, dm >> 16);
                if (__any_sync(0xffffffffu, mx > top || dm > v_top)) {
                    top = fmaxf(top, mx);
                    v_top = max(v_top, __reduce_max_sync(0xffffffffu, dm));
                    // f16 bits e, m: the value is below 2^(e - 14); subnormals below 2^-14
                    v_exp = (int)(v_top >> 10) - 14;
                    const float ref_new = top + (float)(v_exp - 14);
                    const float f = ref == -INFINITY ? 0.0f : kv4_exp2(ref - ref_new);
                    ref = ref_new;
                    l *= f;
#pragma unroll
                    for (int b = 0; b < NB; b++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            o[b][i][0] *= f, o[b][i][1] *= f;
                            if constexpr (PREC) o[b][i][AC - 2] *= f, o[b][i][AC - 1] *= f;
                        }
                }
#pragma unroll
                for (int nb = 0; nb < 4; nb++) {
                    sc[nb][0] = kv4_exp2(sc[nb][0] - ref), sc[nb][1] = kv4_exp2(sc[nb][1] - ref);
                    l += sc[nb][0] + sc[nb][1];
                }
                // ---- O += (P d) (c - 8), 16 positions a step
#pragma unroll
                for (int ks = 0; ks < 2; ks++) {
                    uint32_t ph[NB][2], pl[PREC ? NB : 1][2];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int nb = 2 * ks + e;
                        uint32_t ds[NB];
                        if constexpr (HD == 128) {
                            const uint4 d4 = *reinterpret_cast<const uint4 *>(vscales + (8 * nb + 2 * t4) * 8);
                            ds[0] = d4.x, ds[1] = d4.y, ds[2] = d4.z, ds[3] = d4.w;
                        } else {
                            const uint2 d2 = *reinterpret_cast<const uint2 *>(vscales + (8 * nb + 2 * t4) * 4);
                            ds[0] = d2.x, ds[1] = d2.y;
                        }
#pragma unroll
                        for (int b = 0; b < NB; b++) {
                            const float2 d0 = ka_float2(ds[b / 2]), d1 = ka_float2(ds[NB / 2 + b / 2]);
                            const float x = sc[nb][0] * (b & 1 ? d0.y : d0.x), y = sc[nb][1] * (b & 1 ? d1.y : d1.x);
                            if constexpr (PREC)
                                ka_split(x, y, ph[b][e], pl[b][e]);
                            else
                                ph[b][e] = kv4_half2(x, y);
                        }
                    }
                    uint32_t x0[NB], x1[NB];  // positions 0..7 and 8..15 of the step
                    if constexpr (HD == 128) {
                        const int r = 16 * ks + (lane & 7), b = lane >> 3;
                        ka_ldsm_t(v_at + r * 64 + 16 * (b ^ kv4_turn<128>(r)), x0);
                        ka_ldsm_t(v_at + (r + 8) * 64 + 16 * (b ^ kv4_turn<128>(r + 8)), x1);
                    } else {
                        const int r = 16 * ks + (lane & 7) + 8 * (lane >> 4), b = (lane >> 3) & 1;
                        uint32_t x[4];
                        ka_ldsm_t(v_at + r * 32 + 16 * (b ^ kv4_turn<64>(r)), x);
                        x0[0] = x[0], x0[1] = x[1], x1[0] = x[2], x1[1] = x[3];
                    }
#pragma unroll
                    for (int b = 0; b < NB; b++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {  // dims 32 b + 4 (column) + i; odd i: 16 times the value
                            const uint32_t mask = i & 1 ? 0x00f000f0u : 0x000f000fu;
                            const __half2 off = i & 1 ? off16 : off1;
                            const uint32_t b0 = ka_codes(i & 2 ? x0[b] >> 8 : x0[b], mask, off);
                            const uint32_t b1 = ka_codes(i & 2 ? x1[b] >> 8 : x1[b], mask, off);
                            ka_mma<PREC>(o[b][i], o[b][i], ph[b][0], PREC ? pl[PREC ? b : 0][0] : 0, ph[b][1],
                                         PREC ? pl[PREC ? b : 0][1] : 0, b0, b1);
                        }
                }
            }
            __syncwarp();  // every lane is done with the stage
            if (!dead && filled < mine) {
                fill(filled);
                filled++;
            }
        }
        fills += filled;

        // ---- join the warps: [warp][head][ref, l, o...]
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        __syncthreads();  // the ring is idle
        constexpr int RW = HD + 2;
        float *sums = reinterpret_cast<float *>(ka_smem);
        {
            float *r = sums + (warp * KA_HEADS + gr) * RW;
            if (t4 == 0) r[0] = ref, r[1] = l;
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        float x = o[b][i][e];
                        if constexpr (PREC) x += o[b][i][AC - 2 + e];
                        r[2 + 32 * b + 8 * t4 + 4 * e + i] = i & 1 ? x * 0.0625f : x;
                    }
        }
        __syncthreads();
        const long long first_cta = seg0 / per, last_cta = (seg0 + seen.tiles - 1) / per;
        const bool split = first_cta != last_cta;
        float *mine_out = a.part + ((int64_t)blockIdx.x * 2 + (at == start ? 0 : 1)) * KA_HEADS * RW;
        T *out = reinterpret_cast<T *>(a.out) + (int64_t)tok * a.out_ld + (int64_t)(g * G + h0) * HD;
        // A sum whose reference is still -inf counts only if it is not zero (a NaN, which must come out)
        for (int i = threadIdx.x; i < heads * (HD / 8); i += KA_THREADS) {
            const int h = i / (HD / 8), d = 8 * (i % (HD / 8));
            float top_ref = -INFINITY;
#pragma unroll
            for (int w = 0; w < KA_WARPS; w++) top_ref = fmaxf(top_ref, sums[(w * KA_HEADS + h) * RW]);
            float L = 0.0f, x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < KA_WARPS; w++) {
                const float *r = sums + (w * KA_HEADS + h) * RW;
                if (r[1] == 0.0f) continue;
                const float f = r[0] == -INFINITY ? 1.0f : kv4_exp2(r[0] - top_ref);
                L += f * r[1];
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] += f * r[2 + d + e];
            }
            if (split) {
                float *r = mine_out + h * RW;
                if (d == 0) r[0] = top_ref, r[1] = L;
#pragma unroll
                for (int e = 0; e < 8; e++) r[2 + d + e] = x[e];
            } else {
                const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] *= inv;
                kv4_store_row(out + h * HD + d, x);
            }
        }
        if (split) {
            __threadfence();
            __syncthreads();
            const int expect = (int)(last_cta - first_cta + 1);
            if (threadIdx.x == 0) {
                const int n = atomicAdd(a.arrived + first_cta, 1);
                sh_last = n == expect - 1;
                if (sh_last) a.arrived[first_cta] = 0;
            }
            __syncthreads();
            if (sh_last) {
                __threadfence();
                // run first_cta starts this list at its own start or later (slot 0 or 1); the others at their start
                const int slot0 = seg0 == first_cta * per ? 0 : 1;
                for (int i = threadIdx.x; i < heads * (HD / 8); i += KA_THREADS) {
                    const int h = i / (HD / 8), d = 8 * (i % (HD / 8));
                    float top_ref = -INFINITY;
                    for (int w = 0; w < expect; w++)
                        top_ref = fmaxf(top_ref, __ldcg(a.part + (((first_cta + w) * 2 + (w ? 0 : slot0)) * KA_HEADS + h) * RW));
                    float L = 0.0f, x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                    for (int w = 0; w < expect; w++) {
                        const float *r = a.part + (((first_cta + w) * 2 + (w ? 0 : slot0)) * KA_HEADS + h) * RW;
                        const float2 rl = __ldcg(reinterpret_cast<const float2 *>(r));
                        const float f = rl.y == 0.0f ? 0.0f : rl.x == -INFINITY ? 1.0f : kv4_exp2(rl.x - top_ref);
                        L += f * rl.y;
#pragma unroll
                        for (int e = 0; e < 8; e += 2) {
                            const float2 y = __ldcg(reinterpret_cast<const float2 *>(r + 2 + d + e));
                            x[e] += f * y.x, x[e + 1] += f * y.y;
                        }
                    }
                    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
                    for (int e = 0; e < 8; e++) x[e] *= inv;
                    kv4_store_row(out + h * HD + d, x);
                }
            }
        }
        __syncthreads();  // the sums are read; the ring may be filled again
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        at += n_part;
        if (at == tok0 + (long long)H * seen.tiles) tok0 = at, tok++;
    }
}

// ------------------------------------------------------------------ launchers
template <int HD, typename T>
static cudaError_t rows_launch(bool store, void *k, void *v, int64_t ld, const int32_t *seq, int seq0,
                               const int32_t *pos, int pos0, int64_t n, const Kv4Planes &c, int *err, cudaStream_t st) {
    const dim3 grid((unsigned)((n * (HD / 8) + 255) / 256), 2 * c.n_kv);
    if (store)
        return launch_k(kv4_store_kernel<HD, T>, grid, dim3(256), 0, st, (const T *)k, (const T *)v, ld, seq, seq0, pos,
                        pos0, n, c, err);
    return launch_k(kv4_load_kernel<HD, T>, grid, dim3(256), 0, st, (T *)k, (T *)v, ld, seq, seq0, pos, pos0, n, c, err);
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
    const size_t grid = 2 * (size_t)sm_count, decode = 2 * grid * KA_HEADS * (128 + 2) * 4;
    const size_t prefill = kv4_prefill_part_bytes(sm_count);
    return kv4_counter_bytes(sm_count) + (decode > prefill ? decode : prefill);
}

template <int HD, typename T>
static cudaError_t attn_launch(Kv4Attn &x, const Kv4Planes &c, void *scratch, int sm_count, int *err, cudaStream_t st) {
    using Cfg = Kv4AttnCfg<HD, sizeof(T) == 4>;
    static int set[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!set[dev]) {
        const cudaError_t e =
            cudaFuncSetAttribute(kv4_attn_kernel<HD, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM);
        if (e != cudaSuccess) return e;
        set[dev] = 1;
    }
    // as many CTAs as the most tiles that the cache allows need, at a tile a warp, and at most what is resident
    const int G = x.n_head / c.n_kv, passes = (G + KA_HEADS - 1) / KA_HEADS;
    const int most = x.window > 0 && x.window < c.n_ctx ? x.window + 2 * KA_TILE + x.n_sink : c.n_ctx;
    const int64_t tiles = (int64_t)x.n_tok * c.n_kv * passes * (((most < c.n_ctx ? most : c.n_ctx) + KA_TILE - 1) / KA_TILE);
    const int64_t want = (tiles + KA_WARPS - 1) / KA_WARPS, cap = (int64_t)Cfg::CTAS * sm_count;
    Kv4AttnArgs a;
    a.q = x.q, a.k = x.k, a.v = x.v, a.out = x.out;
    a.q_ld = x.q_ld, a.kv_ld = x.kv_ld, a.out_ld = x.out_ld;
    a.pos = x.pos, a.pos0 = x.pos0, a.seq0 = x.seq0;
    a.n_tok = x.n_tok, a.n_head = x.n_head, a.window = x.window, a.n_sink = x.n_sink, a.scale = x.scale;
    a.arrived = (int *)scratch;
    a.part = kv4_scratch_parts(scratch, sm_count);
    a.err = err;
    return launch_k(kv4_attn_kernel<HD, T>, dim3((unsigned)(want < cap ? want : cap)), dim3(KA_THREADS),
                    (size_t)Cfg::SMEM, st, a, c);
}

cudaError_t launch_kv4_attn(bool f32, int head_dim, Kv4Attn &x, const Kv4Planes &c, void *scratch, int sm_count,
                            int *err, cudaStream_t st) {
    if (x.n_tok <= 0) return cudaSuccess;
    if (head_dim == 128)
        return f32 ? attn_launch<128, float>(x, c, scratch, sm_count, err, st)
                   : attn_launch<128, __nv_bfloat16>(x, c, scratch, sm_count, err, st);
    return f32 ? attn_launch<64, float>(x, c, scratch, sm_count, err, st)
               : attn_launch<64, __nv_bfloat16>(x, c, scratch, sm_count, err, st);
}

}  // namespace tmoe
