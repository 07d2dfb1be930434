// Attention of several sequences at once: what the kernels of attn_few.cu (few query rows) and attn_tc5.cu (chunks and prompts)
// share -- the sequences as the device sees them, the division of the work over the CTAs, and the record of a partial result.
#pragma once

#include "jl_internal.cuh"

// One call. Positions of a sequence are numbered from its first cached one; its new rows are the last `n` of them.
struct AttnMeta;
struct AttnArgs {
    void *out;
    const void *q, *k, *v;
    const int *starts;           // [nseq + 1]
    const int *lens;             // [nseq]; NULL: a sequence is its new rows (packed prompts)
    const int *table;            // [nseq][max_pages]; NULL: position p of sequence s is row starts[s] + p of k and v
    AttnMeta *meta;              // scratch: one of each CTA, then
    float *part;                 // its two partial results
    int *status;                 // [0] code of a wait that ran out, [1] the limit in microseconds
    long long q_tok, q_head;     // strides in elements; the innermost is 1
    long long kv_tok, kv_head, kv_page;
    int nseq, total, hq, hkv, g, d;
    int page_shift, n_pages, max_pages;
    int row_lo, row_hi;          // the launch takes the sequences with row_lo < new rows * g <= row_hi
    int tok_item;                // tokens of one item
    int item_cost, snap;         // units: what an item's start and end take; cuts nearer than this to its end move onto it
    int out_dtype;
    float scale_log2;            // scale * log2(e): softmax is taken to the base 2
};

// first row, new rows, positions readable, position of the first new row; longer than its table?
struct AttnSeq { int row, n, len, pos0, over; };

__host__ __device__ static inline AttnSeq attn_seq(const AttnArgs &a, int s) {
    AttnSeq q;
    int lo = a.starts[s], hi = a.starts[s + 1];
    lo = lo < 0 ? 0 : (lo > a.total ? a.total : lo);
    hi = hi < lo ? lo : (hi > a.total ? a.total : hi);
    q.row = lo;
    q.n = hi - lo;
    int len = a.lens ? a.lens[s] : q.n;
    if (len < 0) len = 0;
    q.pos0 = len - q.n;                           // below zero where a sequence is shorter than its new rows: those see nothing
    q.over = 0;
    if (a.table) {
        const long long cap = (long long)a.max_pages << a.page_shift;
        if (len > cap) {                          // its rows walk the table (and come out NaN); neither pos0 nor a weight passes it
            len = (int)cap;
            q.pos0 = q.pos0 < len ? q.pos0 : len;
            q.over = 1;
        }
    }
    q.len = len;
    const long long rows = (long long)q.n * a.g;
    if (rows <= a.row_lo || rows > a.row_hi) q.n = 0;
    return q;
}
// Positions that the item of tokens [t0, t1) of a sequence walks: those of its last token.
__host__ __device__ static inline int attn_limit(const AttnSeq &q, int t1) {
    const int l = q.pos0 + t1;
    return l < 0 ? 0 : (l > q.len ? q.len : l);
}

// The work is a line of items -- (sequence, block of tok_item tokens, kv head), heads innermost -- and item i is as long on it as
// the positions that it walks plus item_cost units for its start and end. The line is cut into equal shares, one to a CTA,
// the cuts rounded to whole units of positions inside an item; an item that a cut divides leaves a partial result in each CTA,
// and the join (attn.cu) adds them up in ascending order of positions. A few long sequences thus fill the GPU as well as many short
// ones, whatever the lengths, which only the device knows; results depend on the cuts in their rounding and on nothing else.

struct AttnCut { int seq, blk, head, unit; };     // before `unit` of item (seq, blk, head); seq == nseq: the line's end

// a / b of numbers that are not negative: 64-bit division is a long subroutine, and few calls need it.
__host__ __device__ static inline long long attn_div(long long a, long long b) {
    return ((a | b) >> 31) == 0 ? (long long)((unsigned)a / (unsigned)b) : a / b;
}
__host__ __device__ static inline long long attn_item_weight(const AttnSeq &q, int blk, int T, int cost) {
    const int t1 = (blk + 1) * T < q.n ? (blk + 1) * T : q.n;
    return (long long)cost + (q.pos0 > 0 ? q.pos0 : 0) + t1;
}
// Sum of the weights of blocks [0, i) of a sequence, i <= ceil(n / T); for one head.
__host__ __device__ static inline long long attn_blocks_weight(const AttnSeq &q, int i, int T, int cost) {
    if (i <= 0) return 0;
    const long long base = (long long)i * (cost + (q.pos0 > 0 ? q.pos0 : 0));        // no more than a table's 2^30 positions and a cost
    const long long whole = (long long)T * i * (i + 1) / 2;
    const long long over = (long long)i * T - q.n;           // of the last block, if it is the ragged one
    return base + whole - (over > 0 ? over : 0);
}
__host__ __device__ static inline int attn_blocks(const AttnSeq &q, int T) { return (q.n + T - 1) / T; }

// Where a cut at `x` (0 <= x < weight of the sequence times the heads) falls inside sequence s.
__host__ __device__ static inline AttnCut attn_cut_in(const AttnArgs &a, int s, const AttnSeq &q, long long x, int unit_shift, int snap) {
    const int T = a.tok_item, cost = a.item_cost << unit_shift;
    int lo = 0, hi = attn_blocks(q, T) - 1;                  // the last block whose blocks in front weigh no more than x
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (attn_blocks_weight(q, mid, T, cost) * a.hkv <= x) lo = mid; else hi = mid - 1;
    }
    x -= attn_blocks_weight(q, lo, T, cost) * a.hkv;
    const long long w = attn_item_weight(q, lo, T, cost);
    AttnCut c;
    c.seq = s; c.blk = lo; c.head = (int)attn_div(x, w);
    x -= c.head * w;
    const int t1 = (lo + 1) * T < q.n ? (lo + 1) * T : q.n;
    const int units = (attn_limit(q, t1) + (1 << unit_shift) - 1) >> unit_shift;
    long long u = (x - cost + (1 << (unit_shift - 1))) >> unit_shift;
    u = u < 0 ? 0 : (u > units ? units : u);
    if (u <= snap || units - u <= snap) u = 2 * u <= units ? 0 : units;      // a cut this near an item's end would leave a sliver
    c.unit = (int)u;
    return c;
}

// What each CTA left in scratch. A CTA has at most two partial results: slot 0 continues an item that a CTA in front began,
// slot 1 begins an item that the next one continues.
#define ATTN_CONT 1                  // slot 0 holds a part,
#define ATTN_ENDS 2                  // and its item ends in this CTA
#define ATTN_OWN 4                   // slot 1 holds the first part of an item
struct __align__(16) AttnMeta {
    int flags;
    int row, ntok, head;             // of slot 1's item: its first row, its tokens, its kv head
};
__host__ __device__ static inline size_t attn_meta_bytes(int ctas) { return ((size_t)ctas * sizeof(AttnMeta) + 255) & ~(size_t)255; }

// A segment: units [u0, u1) of an item of `units`.
struct AttnSeg { int seq, blk, head, u0, u1, units; AttnSeq q; };

// Walks a CTA's share. first / last are its two cuts.
struct AttnWalk {
    AttnCut at, end;
    AttnSeq q;
    bool fresh;
    __host__ __device__ void begin(const AttnCut &first, const AttnCut &last) { at = first; end = last; fresh = true; }
    // The next segment that has work, or false.
    __host__ __device__ bool next(const AttnArgs &a, int unit_shift, AttnSeg &g) {
        for (;;) {
            if (at.seq >= a.nseq) return false;
            if (fresh) { q = attn_seq(a, at.seq); fresh = false; }
            const int nblk = attn_blocks(q, a.tok_item);
            if (at.blk >= nblk) {                            // past the sequence's last item, or a sequence without rows
                if (at.seq >= end.seq) return false;
                at.seq++; at.blk = at.head = at.unit = 0; fresh = true;
                continue;
            }
            const bool last = at.seq == end.seq && at.blk == end.blk && at.head == end.head;
            const int t1 = (at.blk + 1) * a.tok_item < q.n ? (at.blk + 1) * a.tok_item : q.n;
            g.units = (attn_limit(q, t1) + (1 << unit_shift) - 1) >> unit_shift;
            g.seq = at.seq; g.blk = at.blk; g.head = at.head; g.q = q;
            g.u0 = at.unit;
            g.u1 = last ? end.unit : g.units;
            const bool some = g.u0 < g.u1 || (g.units == 0 && !last);
            if (last) at.seq = a.nseq;                       // nothing after it
            else {
                at.unit = 0;
                if (++at.head == a.hkv) { at.head = 0; at.blk++; }
            }
            if (some) return true;
        }
    }
};

__host__ __device__ static inline long long attn_seq_weight(const AttnArgs &a, const AttnSeq &q, int unit_shift) {
    return attn_blocks_weight(q, attn_blocks(q, a.tok_item), a.tok_item, a.item_cost << unit_shift) * a.hkv;
}
// The shares of a line of `total`: how many there are (each min_units units at least), where share `cta` lies, and how near an item's
// end a cut snaps onto it. False: the CTA has no share.
__host__ __device__ static inline bool attn_cuts(long long total, int cta, int grid, int unit_shift, int min_units, int most, long long &b0,
                                                 long long &b1, int &snap) {
    long long ctas = attn_div(total, (long long)min_units << unit_shift);
    ctas = ctas < 1 ? 1 : (ctas > grid ? grid : ctas);
    if (total == 0 || cta >= ctas) return false;
    const long long share = attn_div(total, ctas), rest = total - share * ctas;       // total * cta may pass 63 bits
    b0 = share * cta + attn_div(rest * cta, ctas);
    b1 = share * (cta + 1) + attn_div(rest * (cta + 1), ctas);
    const long long quarter = share >> (unit_shift + 2);
    snap = quarter < most ? (int)quarter : most;
    return true;
}
static inline void attn_share_host(const AttnArgs &a, int cta, int grid, int unit_shift, int min_units, AttnCut &first, AttnCut &last) {
    long long total = 0, b0, b1, base = 0;
    int snap;
    for (int s = 0; s < a.nseq; ++s) total += attn_seq_weight(a, attn_seq(a, s), unit_shift);
    first = last = AttnCut{a.nseq, 0, 0, 0};
    if (!attn_cuts(total, cta, grid, unit_shift, min_units, a.snap, b0, b1, snap)) return;
    for (int s = 0; s < a.nseq; ++s) {
        const AttnSeq q = attn_seq(a, s);
        const long long w = attn_seq_weight(a, q, unit_shift);
        if (b0 >= base && b0 < base + w) first = attn_cut_in(a, s, q, b0 - base, unit_shift, snap);
        if (b1 >= base && b1 < base + w) last = attn_cut_in(a, s, q, b1 - base, unit_shift, snap);
        base += w;
    }
}

#ifdef __CUDACC__
// The two cuts of CTA `cta` of `grid`, found by each warp; every lane returns them. The sequences are gone over twice, for the
// line's length and for the cuts' places; the first 128 are fetched once, all at a time (a pass of dependent loads is 0.8 us).
__device__ static inline void attn_share(const AttnArgs &a, int cta, int grid, int unit_shift, int min_units, AttnCut &first, AttnCut &last) {
    constexpr int KEPT = 4;
    const int lane = threadIdx.x & 31;
    AttnSeq kept[KEPT];
    long long weight[KEPT], total = 0;
#pragma unroll
    for (int c = 0; c < KEPT; ++c) {
        kept[c] = AttnSeq{0, 0, 0, 0, 0};
        if (c * 32 + lane < a.nseq) kept[c] = attn_seq(a, c * 32 + lane);
    }
#pragma unroll
    for (int c = 0; c < KEPT; ++c) total += weight[c] = attn_seq_weight(a, kept[c], unit_shift);       // zero for none
    for (int s0 = KEPT * 32; s0 < a.nseq; s0 += 32)
        if (s0 + lane < a.nseq) total += attn_seq_weight(a, attn_seq(a, s0 + lane), unit_shift);
#pragma unroll
    for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    first.seq = last.seq = a.nseq;
    first.blk = first.head = first.unit = last.blk = last.head = last.unit = 0;
    long long b0, b1, base = 0;
    int snap;
    if (!attn_cuts(total, cta, grid, unit_shift, min_units, a.snap, b0, b1, snap)) return;
    auto look = [&](int s0, const AttnSeq &q, long long w) {
        long long upto = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const long long from = base + upto - w;
        base += __shfl_sync(0xffffffffu, upto, 31);
        const unsigned m0 = __ballot_sync(0xffffffffu, b0 >= from && b0 < from + w), m1 = __ballot_sync(0xffffffffu, b1 >= from && b1 < from + w);
        auto place = [&](unsigned m, long long b, AttnCut &to) {
            if (!m) return;
            AttnCut c = {a.nseq, 0, 0, 0};
            if ((m >> lane) & 1) c = attn_cut_in(a, s0 + lane, q, b - from, unit_shift, snap);
            const int l = __ffs(m) - 1;
            to.seq = __shfl_sync(0xffffffffu, c.seq, l); to.blk = __shfl_sync(0xffffffffu, c.blk, l);
            to.head = __shfl_sync(0xffffffffu, c.head, l); to.unit = __shfl_sync(0xffffffffu, c.unit, l);
        };
        place(m0, b0, first);
        place(m1, b1, last);
    };
#pragma unroll
    for (int c = 0; c < KEPT; ++c)
        if (c * 32 < a.nseq && base <= b1) look(c * 32, kept[c], weight[c]);
    for (int s0 = KEPT * 32; s0 < a.nseq && base <= b1; s0 += 32) {
        AttnSeq q = {0, 0, 0, 0, 0};
        if (s0 + lane < a.nseq) q = attn_seq(a, s0 + lane);
        look(s0, q, attn_seq_weight(a, q, unit_shift));
    }
}

// Two results as out_dtype, from row-major element offset `at` (even).
__device__ __forceinline__ void attn_store2(void *out, int dtype, size_t at, float x, float y) {
    if (dtype == JL_DT_F32) *reinterpret_cast<float2 *>(static_cast<float *>(out) + at) = make_float2(x, y);
    else if (dtype == JL_DT_BF16) *reinterpret_cast<__nv_bfloat162 *>(static_cast<__nv_bfloat16 *>(out) + at) = __floats2bfloat162_rn(x, y);
    else *reinterpret_cast<__half2 *>(static_cast<__half *>(out) + at) = __floats2half2_rn(x, y);
}
__device__ __forceinline__ void attn_store4(void *out, int dtype, size_t at, float4 v) {
    if (dtype == JL_DT_F32) {
        *reinterpret_cast<float4 *>(static_cast<float *>(out) + at) = v;
        return;
    }
    uint2 w;
    if (dtype == JL_DT_BF16) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
        w = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
    } else {
        const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
        w = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
    }
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(out) + at) = w;
}
#endif

// A partial result in scratch: [rows][d] weighted sums of V, then [rows] maxima (base 2, scaled), then [rows] sums, all f32. A row that sees
// nothing has the maximum -inf and the sum 0, and its result is zero. One that sees positions whose scores are all -inf has the maximum
// -inf too, but no result (0 / 0): its sum is ATTN_DARK, which no part's weight multiplies, and if no part has more, its result is NaN.
#define ATTN_DARK (-1.f)
__host__ __device__ static inline size_t attn_slot_floats(int rows, int d) { return (size_t)rows * (d + 2); }
#define ATTN_FEW_ROWS 16
#define ATTN_FEW_CTAS 3          // to an SM
#define ATTN_FEW_MAX 512         // in all: the join keeps 64 parts to each of eight warps
#define ATTN_TC_ROWS 256         // or 128, and twice the CTAs

// Launched so that the kernel may be put in place while the one in front of it in the stream drains (unless the context is to do without).
template <typename... P, typename... Args>
static cudaError_t attn_launch_pdl(const jl_ctx *ctx, void (*kern)(P...), dim3 grid, dim3 block, int smem, cudaStream_t s, Args... args) {
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = block; cfg.dynamicSmemBytes = smem; cfg.stream = s; cfg.attrs = at;
    cfg.numAttrs = (ctx->opts.flags & JL_FLAG_NO_PDL) ? 0 : 1;
    return cudaLaunchKernelEx(&cfg, kern, static_cast<P>(args)...);
}

// attn_few.cu, attn_tc5.cu, attn.cu
int attn_launch_few(jl_ctx *ctx, const AttnArgs &a, int dtype, cudaStream_t s);
// max_rows: query rows of a sequence and kv head, at most
int attn_launch_tc5(jl_ctx *ctx, const AttnArgs &a, int dtype, long long max_rows, cudaStream_t s);
// unit: positions below which no cut divides an item
int attn_launch_merge(jl_ctx *ctx, const AttnArgs &a, int rows, int ctas, int unit, cudaStream_t s);
static inline int attn_few_grid(const jl_ctx *ctx) {
    return ctx->sm_count * ATTN_FEW_CTAS < ATTN_FEW_MAX ? ctx->sm_count * ATTN_FEW_CTAS : ATTN_FEW_MAX;
}
