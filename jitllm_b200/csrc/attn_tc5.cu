// Attention for many query rows (chunks of new tokens, prompts) on tcgen05.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(scale log2(e) q.k_j - m),  m a maximum of the exponents so far
//
// An item is 256 query rows of one kv head in two tiles of 128 (or one tile: TaRoles): (new token, query head of the group),
// token-major, so that grouped heads share the tile's keys and a causal edge is 128 / g tokens wide. Per 128 positions a tile takes two
// 128 x 128 x d products (tcgen05.mma, kind::f16: S = Q K^T out of shared memory, O += P V with P out of TMEM; 512 clocks each at d = 128)
// and 128 x 128 exponentials (1024 clocks of the exponential unit). TMEM holds S and O of both tiles and nothing else, P goes over S: so a
// tile's softmax and products follow one another, and the two tiles alternate, one on the tensor core while the other's softmax runs.
//
// Roles of a CTA: a softmax warpgroup to a tile (a thread owns a row: S comes to its registers, P goes back over S's columns, 16 bits);
// a warp each that issues the products, that loads (K and V tiles of 128 positions through one ring by TMA, a box to a page and 64
// columns; Q once an item), that looks over the V tiles at a sequence's edge, and that walks the CTA's share.
//
// An f32 result takes a weight as two f16 values or three bf16 values (S's columns hold two: the third goes over the first once the product
// with that is done, while the product with the second runs), to a maximum that is looked for. A third more products: bf16, five tokens of
// 32 sequences 72 us (two parts: 60), a prompt of 1531 tokens 71 (67), of 16,384 3750 (2635); errors 1e-7 to 8e-7 of relative rms up to
// 1500 positions, 8e-7 to 2e-6 with two. Both tiles' first parts in front of both thirds: 4430 us, the tiles fall into step.
//
// What bounds it: a tile's round of 128 positions, 1450 clocks of softmax (1290 of a loop of nothing else, of them 1024 exponentials), 300
// for S, P and the barriers to change hands, 1024 of products: 3250 clocks as counted with two tiles at work, where the tensor core
// alone would need 2048. Tried and not kept: exponentials on the FMA pipe by a polynomial (it costs the scheduler what it saves the other
// unit), rows split over two warps (the exchange of their maxima costs as much), S in halves of 64 positions with columns of their own
// (the products S = Q K^T then read Q twice as often and take 1.5 times as long), an MMA warp to a tile (their products run side by side
// and the tiles fall into step), masked tiles on the short way (a second copy of it: registers spill, every case is 3 to 8 % slower).
// A 16,384-token prompt of 32 heads over 8: 2.05 to 2.1 ms, 1.05 to 1.08 PFLOP/s, at the clock that the power limit leaves (1.8 ms in the
// first moments of a cool GPU). Short prompts are bound by their
// items' ends: a 1531-token one spends 2 x 10,000 of a CTA's 70,000 clocks on them (7000 on the rows' way out, the rest on masks).
#include "attn.cuh"
#include "tc5.cuh"

#define TA_UNIT_SHIFT 7
#define TA_KV 128                        // positions of a unit
// A CTA's warps: four to a tile of 128 rows for the softmax, then one each for the products, the loads, the edges and the walk. Two tiles
// to a CTA and an SM where there are rows enough (they share K and V); else one tile, and two CTAs to an SM: a tile's softmax and products
// follow one another, and only another tile's work fills the gaps.
template <int TILES> struct TaRoles {
    static constexpr int SOFT = 4 * TILES, MMA = SOFT, PRODUCER = SOFT + 1, EDGES = SOFT + 2, WALK = SOFT + 3, WARPS = SOFT + 4;
    static constexpr int CTAS = TILES == 1 ? 2 : 1, ROWS = 128 * TILES;
    // Registers a thread: launched with 168 (384 threads) or 128 (256); the softmax warpgroups, whose rows of S and P live in registers, go
    // up by 40 (256 threads: 10240) or 72 (128 threads: 9216), the last one goes down by 80 or 72 (128 threads).
    static constexpr int REGS_SOFT = TILES == 1 ? 200 : 208, REGS_OTHER = TILES == 1 ? 56 : 88;
};
#define TA_STATUS_CODE 7
// What an item's start and end take against a unit: Q's arrival, the first S, the last product, the rows' way out; 10,000 clocks beside
// 3250 of two tiles, 6000 beside 2900 of one. With 1, 2, 3 and 4 a prompt of 16,384 tokens takes 2270, 2020, 1875 and 1865 us, 24 prompts of 1
// to 1900 tokens 72, 61.5, 60.8 and 65, one of 1531 52, 48.5, 50.5 and 49 (how the cuts happen to fall). One tile, 1, 2 and 3: 49.5, 48
// and 47.5 us for five tokens of 32 sequences.
#define TA_ITEM_COST 3
#define TA_ITEM_COST_ONE 2
// Two tiles: a cut one unit from an item's end moves onto it. The sliver that it saves costs its CTA 10,000 clocks; a cut further off,
// moved, would cost the CTA next to it more (24 packed prompts 61.1 us with none, 60.8 with one unit, 62.6 with two; 1531 tokens 49.8, 50.5,
// 50.2). One tile has less to save: the same with none and with one.
#define TA_SNAP 1
// One tile up to as many rows as it has (five tokens of 8 heads: 48 us against 55 with a second tile idle); beyond, two: a 1531-token
// prompt takes 50.5 us so and 58 as single tiles, whose CTAs load K and V each for itself.
#define TA_ONE_TILE_ROWS 128
// log2 of a weight at the reference, and the limit of a tile's sum of weights. f16 ends at 2^-24 and at 65504: with weights of one at the
// reference a long flat tail below 2^-25 of it would leave the products but not the sum (131,071 positions: 0.4 % of a result). At 2^6 a
// weight is held to 2^-31 and may still grow by 2^10 over the reference; at 2^8 more tiles pass the limit (f16, 24 packed prompts 63.2 us
// against 60.3, one of 1531 tokens 52.4 against 48.7). f32 results take the weights to a maximum that is known, and so to 2^14.
template <bool BF16, bool HILO> struct TaWeights {
    static constexpr float LOG_TOP = BF16 ? 0.f : HILO ? 14.f : 6.f, LIMIT = BF16 ? 16384.f : 65504.f;
    static constexpr float ROOM = BF16 ? 14.f : 1.f;         // log2 of what a weight of an f32 result may pass 2^LOG_TOP by
};

// The bounded wait of this kernel's roles. A try that may sleep for up to 20 us: the warps that wait are many, and their polling would take
// the issue slots of those that work.
// A patient role's wait spans others' whole work -- all of a segment, or the walk over the sequences -- and so has 4096 times the limit, up to
// ten seconds more than it. Those others give up first where something is lost, and end it.
#define TA_PATIENCE 4096ull
#define TA_PATIENCE_NS 10000000000ull
// What is waited for at a CTA's end, whatever the limit is: copies and products that are on their way end by themselves.
#define TA_DRAIN_NS 1000000000ull
__device__ __forceinline__ bool ta_wait(uint32_t bar, uint32_t parity, volatile int *abort_flag, bool patient = false) {
    uint64_t t0 = 0;
    for (;;) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(bar), "r"(parity), "r"(20000u)
            : "memory");
        if (done) return true;
        if (*abort_flag) return false;
        const uint64_t t = jl_gtime_ns();
        if (!t0) t0 = t;
        else {
            const uint64_t limit = tc5_limit_ns(abort_flag);
            if (t - t0 > limit + (patient ? min((unsigned long long)limit * (TA_PATIENCE - 1), TA_PATIENCE_NS) : 0ull)) break;
        }
    }
    *abort_flag = 1;
    return false;
}
// D[tmem] (+)= A[tmem] * B[smem desc].
__device__ __forceinline__ void ta_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void ta_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
        "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
        "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void ta_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
// The loads into r are complete. The registers are operands, so that nothing that reads them moves in front of the wait.
__device__ __forceinline__ void ta_wait_ld(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                 "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                 "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]),
                 "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void ta_wait_ld(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                 "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void ta_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void ta_tma_3d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void ta_tma_4d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, int w, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
                 : "memory");
}
// V tile as the B operand, N (the head's columns) contiguous: 64-column halves 16 KB apart, groups of 8 positions 1 KB apart.
__device__ __forceinline__ uint64_t ta_desc_mn(uint32_t smem_addr) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr >> 4) & 0x3FFF);
    d |= (uint64_t)((128 * 128) >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
__device__ __forceinline__ float ta_max(float x, float y) {          // NaN if either is
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(x), "f"(y));
    return m;
}
// d += x on both halves.
__device__ __forceinline__ void ta_add2(float (&d)[2], float x, float y) {
    asm("{\n\t.reg .b64 rd, rx;\n\t"
        "mov.b64 rd, {%0, %1};\n\t"
        "mov.b64 rx, {%2, %3};\n\t"
        "add.rn.f32x2 rd, rd, rx;\n\t"
        "mov.b64 {%0, %1}, rd;\n\t}"
        : "+f"(d[0]), "+f"(d[1])
        : "f"(x), "f"(y));
}
__device__ __forceinline__ float ta_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <bool BF16> __device__ __forceinline__ uint32_t ta_pack(float x, float y) {
    if constexpr (BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __half2 h = __floats2half2_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}
template <bool BF16> __device__ __forceinline__ float2 ta_unpack(uint32_t w) {
    if constexpr (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    else return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
// A packed pair with what is infinite or NaN in it set to zero.
template <bool BF16> __device__ __forceinline__ uint32_t ta_finite(uint32_t w) {
    constexpr uint32_t E = BF16 ? 0x7F80u : 0x7C00u;
    if ((w & E) == E) w &= 0xFFFF0000u;
    if ((w & (E << 16)) == (E << 16)) w &= 0x0000FFFFu;
    return w;
}

// What the roles need of a segment. One warp walks the CTA's share and hands the segments out through a ring in shared memory: a row of S
// fills most of a softmax thread's registers, and a walk of its own would spill the rest.
struct __align__(16) TaSeg {
    int seq, head;               // seq < 0: the share's end
    int u0, u1, whole;           // units; is this all of the item?
    int ends;                    // the item ends here
    int tok0, ntok;              // of the item, in the sequence
    int e[2];                    // units of the segment that each tile walks
    int edge;                    // units from this one on hold positions that some row of the item does not see, or the sequence's end
    int row, n, len, pos0, over; // of the sequence
};
#define TA_SEGS 4
template <int TILES>
__device__ __forceinline__ void ta_seg(const AttnArgs &a, const AttnSeg &g, volatile TaSeg *t) {
    const int tq = a.tok_item / TILES, tok0 = g.blk * a.tok_item;
    t->seq = g.seq; t->head = g.head; t->u0 = g.u0; t->u1 = g.u1;
    t->whole = g.u0 == 0 && g.u1 == g.units;
    t->ends = g.u1 == g.units;
    t->tok0 = tok0;
    t->ntok = min(a.tok_item, g.q.n - tok0);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int first = tok0 + i * tq;
        const int units = i < TILES && first < g.q.n ? (attn_limit(g.q, min(first + tq, g.q.n)) + TA_KV - 1) >> TA_UNIT_SHIFT : 0;
        t->e[i] = max(0, min(units, g.u1) - g.u0);
    }
    t->edge = min(attn_limit(g.q, tok0 + 1), g.q.len) >> TA_UNIT_SHIFT;
    t->row = g.q.row; t->n = g.q.n; t->len = g.q.len; t->pos0 = g.q.pos0; t->over = g.q.over;
}
__device__ __forceinline__ int ta_seen(const volatile TaSeg *t, int tok1) {          // attn_limit
    return max(0, min(t->pos0 + tok1, t->len));
}

template <int D, int TILES> struct TaSmem {
    static constexpr int NH = D / 64;                         // 64-column halves: 128 bytes of a row, the swizzle's width
    static constexpr int HALF = 128 * 128;                    // bytes of 128 rows of one
    static constexpr int TILE = NH * HALF;
    static constexpr int STAGES = (D == 128 ? 2 : 4) * TILES;
    static constexpr int PASS = D == 128 && TILES == 1 ? 64 : 128;       // bytes of a row that leave at a time
    static constexpr int Q = 0, KV = TILES * TILE, OUT = KV + STAGES * TILE, BARS = OUT + 4 * TILES * 32 * PASS;     // OUT: 32 rows of PASS bytes to a softmax warp
    // barriers: kv_full[STAGES], kv_empty[STAGES], q_full, q_empty, s_full[2], p_full[2], o_full[2], drain, v_ok[OKS], e_full[OKS], g_full[TA_SEGS], g_empty[TA_SEGS], h_used[2]
    static constexpr int OKS = D == 128 ? 4 : 8;              // more than the V tiles that the ring can hold
    static constexpr int NBARS = 2 * STAGES + 11 + 2 * OKS + 2 * TA_SEGS;
    static constexpr int SEGS = (BARS + NBARS * 8 + 15) & ~15;
    static constexpr int MISC = SEGS + TA_SEGS * (int)sizeof(TaSeg);      // tmem address, abort flag and limit, seg_bad[4], seg_odd[4]
    static constexpr int TOTAL = MISC + 64 + 1024;           // 1024: the tiles start on a swizzle atom
};

// A row's results get back what the edge warp took out of positions [p0, p1), which the row sees. The row is `dtype` at dst.
template <bool BF16>
__device__ __noinline__ void ta_odd(const AttnArgs *a, int seq, int head, int row, int p0, int p1, void *dst, int dtype) {
    for (int p = p0; p < p1; ++p) {
        long long at;
        if (a->table) {
            const int page = a->table[(long long)seq * a->max_pages + (p >> a->page_shift)];
            if ((unsigned)page >= (unsigned)a->n_pages) continue;
            at = page * a->kv_page + head * a->kv_head + (p & ((1 << a->page_shift) - 1)) * a->kv_tok;
        } else {
            at = (long long)(row + p) * a->kv_tok + head * a->kv_head;
        }
        const uint32_t *v = reinterpret_cast<const uint32_t *>(static_cast<const uint16_t *>(a->v) + at);
#pragma unroll 1
        for (int y = 0; y < a->d / 2; ++y) {
            const uint32_t w = v[y];                         // a plain load: the kernel in front may have written it (attn_few.cu)
            if (ta_finite<BF16>(w) == w) continue;
            float2 f = ta_unpack<BF16>(w);                   // what is finite of the pair is in the sum already
            f.x = isfinite(f.x) ? 0.f : f.x;
            f.y = isfinite(f.y) ? 0.f : f.y;
            if (dtype == JL_DT_F32) {
                float *o = static_cast<float *>(dst) + 2 * y;
                o[0] += f.x; o[1] += f.y;
            } else if (dtype == JL_DT_BF16) {
                __nv_bfloat16 *o = static_cast<__nv_bfloat16 *>(dst) + 2 * y;
                o[0] = __float2bfloat16(__bfloat162float(o[0]) + f.x); o[1] = __float2bfloat16(__bfloat162float(o[1]) + f.y);
            } else {
                __half *o = static_cast<__half *>(dst) + 2 * y;
                o[0] = __float2half(__half2float(o[0]) + f.x); o[1] = __float2half(__half2float(o[1]) + f.y);
            }
        }
    }
}

template <int D, int TILES, bool BF16, bool HILO>
__global__ void __launch_bounds__(TaRoles<TILES>::WARPS * 32, TaRoles<TILES>::CTAS)
attn_tc5_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                const __grid_constant__ CUtensorMap vmap, int box_rows, int min_units) {
    using L = TaSmem<D, TILES>;
    using R = TaRoles<TILES>;
    using W = TaWeights<BF16, HILO>;
    constexpr bool THIRD = BF16 && HILO;                    // a weight has three parts; the third goes over the first once that is used
    constexpr int TM_O = TILES * 128;                       // O's columns in TMEM, behind S's
    extern __shared__ uint8_t raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t sbase = smem_u32(smem), bars = sbase + L::BARS;
    const uint32_t kv_full = bars, kv_empty = bars + 8 * L::STAGES, q_full = bars + 16 * L::STAGES, q_empty = q_full + 8, s_full = q_full + 16,
                   p_full = q_full + 32, o_full = q_full + 48, drain = q_full + 64, v_ok = q_full + 72, e_full = v_ok + 8 * L::OKS, g_full = e_full + 8 * L::OKS,
                   g_empty = g_full + 8 * TA_SEGS, h_used = g_empty + 8 * TA_SEGS;
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(smem + L::MISC);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::MISC + 4);        // [0] flag, [1] limit
    volatile int *seg_bad = reinterpret_cast<volatile int *>(smem + L::MISC + 16), *seg_odd = seg_bad + 4;
    const int warp = tc5_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int tq = a.tok_item / TILES;
    if (threadIdx.x == 0) {
        for (int s = 0; s < L::STAGES; ++s) { mbar_init(kv_full + 8 * s, 1); mbar_init(kv_empty + 8 * s, 1); }
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(s_full + 8 * i, 1);
            mbar_init(p_full + 8 * i, 4);                   // one arrival a softmax warp
            mbar_init(o_full + 8 * i, 1);
            mbar_init(h_used + 8 * i, 1);
        }
        for (int i = 0; i < 2 * L::OKS; ++i) mbar_init(v_ok + 8 * i, 1);       // and e_full
        for (int i = 0; i < TA_SEGS; ++i) { mbar_init(g_full + 8 * i, 1); mbar_init(g_empty + 8 * i, R::SOFT + 3); }     // all but the walk
        mbar_init(drain, 1);
        for (int i = 0; i < 4; ++i) seg_bad[i] = seg_odd[i] = 0;
        abort_flag[0] = 0;
        abort_flag[1] = a.status[1];
        mbar_init_fence();
    }
    if (warp == R::MMA) tc5_alloc(smem_u32(const_cast<uint32_t *>(tmem_slot)), 256 * TILES);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    tc5_fence_before();
    __syncthreads();
    tc5_fence_after();
    const uint32_t tmem = *tmem_slot;                       // S of the tiles at columns 0, 128; O behind them
    volatile TaSeg *const ring = reinterpret_cast<volatile TaSeg *>(smem + L::SEGS);
    bool ok = true;
    uint32_t gi = 0;                                        // segments seen
    // the next segment, or NULL at the end of the share
    auto seg_next = [&]() -> const volatile TaSeg * {
        ok = ok && __all_sync(0xffffffffu, ta_wait(g_full + 8 * (gi % TA_SEGS), (gi / TA_SEGS) & 1, abort_flag, true));
        const volatile TaSeg *t = ring + gi % TA_SEGS;
        return ok && t->seq >= 0 ? t : nullptr;
    };
    auto seg_done = [&]() {
        __syncwarp();
        if (lane == 0) mbar_arrive(g_empty + 8 * (gi % TA_SEGS));
        gi++;
    };
#define TA_REGS(how, n) asm volatile("setmaxnreg." how ".sync.aligned.u32 %0;" ::"n"(n))

    if (warp == R::PRODUCER) {
        TA_REGS("dec", R::REGS_OTHER);
        // ------------------------------------------------ producer: the ring's tiles are K's and V's in turn
        const uint32_t sb = (uint32_t)tc5_uniform((int)sbase);
        uint32_t it = 0, segs = 0, edges = 0;               // tiles issued, segments with work, edge tiles of V
        const bool leader = tc5_elect();
        while (const volatile TaSeg *t = seg_next()) {
            const int u0 = tc5_uniform(t->u0), E = tc5_uniform(max(t->e[0], t->e[1]));
            if (E == 0) { seg_done(); continue; }
            const int u1 = u0 + E, len = tc5_uniform(t->len), head = tc5_uniform(t->head), row = tc5_uniform(t->row), edge = tc5_uniform(t->edge);
            const int *table = a.table ? a.table + (long long)t->seq * a.max_pages : nullptr;
            if (segs) ok = __all_sync(0xffffffffu, ta_wait(q_empty, (segs - 1) & 1, abort_flag));
            if (!ok) break;
            const int tiles = tc5_uniform(t->ntok > tq ? 2 : 1), tok = row + tc5_uniform(t->tok0);
            if (leader) {
                seg_bad[segs & 3] = t->over;
                mbar_arrive_expect_tx(q_full, tiles * L::NH * a.g * tq * 128);       // boxes of g heads x tq tokens x 64 columns
                for (int i = 0; i < tiles; ++i)
#pragma unroll
                    for (int h = 0; h < L::NH; ++h)
                        ta_tma_3d(sb + L::Q + i * L::TILE + h * L::HALF, &qmap, h * 64, head * a.g, tok + i * tq, q_full);
            }
            __syncwarp();
            const int nbox = TA_KV / box_rows;               // a page, or the part of it in a unit; lane b looks up the page of box b
            auto page_of = [&](int u) -> int {
                const int p = u * TA_KV + lane * box_rows;
                return table && lane < nbox && u < u1 && p < len ? table[p >> a.page_shift] : 0;
            };
            int page = page_of(u0);
            for (int u = u0; u < u1 && ok; ++u) {
                const int boxes = min(nbox, (len - u * TA_KV + box_rows - 1) / box_rows);
                int z = page;
                if (table && (unsigned)z >= (unsigned)a.n_pages) {           // out of the map: zeros
                    z = a.n_pages;
                    seg_bad[segs & 3] = 1;
                }
                page = page_of(u + 1);
                const int y = table ? (u * TA_KV) & ((1 << a.page_shift) - 1) : row + u * TA_KV;
#pragma unroll
                for (int kv = 0; kv < 2 && ok; ++kv, ++it) {
                    const uint32_t s = it % L::STAGES;
                    if (it >= (uint32_t)L::STAGES) ok = __all_sync(0xffffffffu, ta_wait(kv_empty + 8 * s, (it / L::STAGES + 1) & 1, abort_flag));
                    if (!ok) break;
                    // an edge tile of V lands on a barrier of its own, which the edge warp waits for: it sees no other tile, and a
                    // stage's barrier would look to it as if a fill that it has not seen were the one it wants
                    uint32_t full = kv_full + 8 * s;
                    if (kv && u >= edge) {
                        if (leader) mbar_arrive(full);
                        full = e_full + 8 * (edges++ % L::OKS);
                    }
                    if (leader) mbar_arrive_expect_tx(full, boxes * L::NH * box_rows * 128);
                    uint32_t dst = sb + L::KV + s * L::TILE;
                    for (int b = 0; b < boxes; ++b, dst += box_rows * 128) { // one lane issues: its operands are the same in every lane
                        const int zb = __shfl_sync(0xffffffffu, z, b);
                        if (leader) {
#pragma unroll
                            for (int h = 0; h < L::NH; ++h) ta_tma_4d(dst + h * L::HALF, kv ? &vmap : &kmap, h * 64, y, head, zb, full);
                        }
                    }
                    __syncwarp();
                }
            }
            segs++;
            seg_done();
        }
        // A copy must not outlive its CTA: the last on each barrier are waited for here. Where all went well they have landed or are about to;
        // where a role gives up, perhaps after this one is done, nobody else waits for them.
        if (segs) mbar_wait_ns(q_full, (segs - 1) & 1, TA_DRAIN_NS);
        for (uint32_t i = it > (uint32_t)L::STAGES ? it - L::STAGES : 0; i < it; ++i)
            mbar_wait_ns(kv_full + 8 * (i % L::STAGES), (i / L::STAGES) & 1, TA_DRAIN_NS);
        for (uint32_t i = edges > (uint32_t)L::OKS ? edges - L::OKS : 0; i < edges; ++i)
            mbar_wait_ns(e_full + 8 * (i % L::OKS), (i / L::OKS) & 1, TA_DRAIN_NS);
    } else if (warp == R::MMA) {
        TA_REGS("dec", R::REGS_OTHER);
        // ------------------------------------------------ products
        constexpr uint32_t type = BF16 ? (1u << 7) | (1u << 10) : 0u;
        constexpr uint32_t id_s = tc5_idesc(128, 128) | type, id_o = tc5_idesc(128, D) | type | (1u << 16);   // V: N contiguous
        const bool leader = tc5_elect();
        // What the instructions take has to be known to be the same in every lane: otherwise each operand of each is moved to a uniform
        // register on its own, and a product takes longer to issue than to run (95 clocks against 60).
        const uint32_t tm = (uint32_t)tc5_uniform((int)tmem), sb = (uint32_t)tc5_uniform((int)sbase);
        const uint64_t qd = tc5_smem_desc(sb + L::Q), kd = tc5_smem_desc(sb + L::KV), vd = ta_desc_mn(sb + L::KV);
        uint32_t it = 0, segs = 0, done[2] = {0, 0}, edges = 0;      // tiles of the ring consumed, segments, P tiles consumed, edge tiles
        auto scores = [&](int i, uint32_t stage) {                   // S of tile i = Q K^T
            const uint64_t q = qd + i * (L::TILE >> 4), k = kd + stage * (L::TILE >> 4);
#pragma unroll
            for (int x = 0; x < D / 16; ++x)
                tc5_mma_f16(tm + i * 128, q + ((x / 4) * (L::HALF >> 4) + 2 * (x % 4)), k + ((x / 4) * (L::HALF >> 4) + 2 * (x % 4)), id_s, x != 0);
            tc5_commit(s_full + 8 * i);
        };
        while (const volatile TaSeg *t = seg_next()) {
            const int u0 = tc5_uniform(t->u0), e0 = tc5_uniform(t->e[0]), e1 = tc5_uniform(t->e[1]), E = max(e0, e1);
            if (E == 0) { seg_done(); continue; }
            const int edge = tc5_uniform(t->edge) - u0;
            ok = __all_sync(0xffffffffu, ta_wait(q_full, segs & 1, abort_flag)) &&
                 __all_sync(0xffffffffu, ta_wait(kv_full + 8 * (it % L::STAGES), (it / L::STAGES) & 1, abort_flag));
            if (!ok) break;
            tc5_fence_after();
            if (leader) {
                if (e0 > 0) scores(0, it % L::STAGES);
                if (e1 > 0) scores(1, it % L::STAGES);
                tc5_commit(kv_empty + 8 * (it % L::STAGES));
                if (E == 1) tc5_commit(q_empty);
            }
            it++;                                                    // now at V of unit 0
            for (int j = 0; j < E && ok; ++j, it += 2) {
                const uint32_t sv = it % L::STAGES, sk = (it + 1) % L::STAGES;
                if (j >= edge) {
                    ok = __all_sync(0xffffffffu, ta_wait(v_ok + 8 * (edges % L::OKS), (edges / L::OKS) & 1, abort_flag));
                    edges++;
                } else {
                    ok = __all_sync(0xffffffffu, ta_wait(kv_full + 8 * sv, (it / L::STAGES) & 1, abort_flag));
                }
                if (ok && j + 1 < E) ok = __all_sync(0xffffffffu, ta_wait(kv_full + 8 * sk, ((it + 1) / L::STAGES) & 1, abort_flag));
                const uint64_t v = vd + sv * (L::TILE >> 4);
                // O of tile i += P V, P's first part and (HILO) second, or its third; with the last part S of the next unit, or the segment's end
                auto product = [&](int i, bool first, bool last) {
                    const int e = i ? e1 : e0;
                    if (!ok || j >= e) return;
                    ok = __all_sync(0xffffffffu, ta_wait(p_full + 8 * i, done[i] & 1, abort_flag));
                    if (!ok) return;
                    tc5_fence_after();
                    if (leader) {
                        const uint32_t p = tm + i * 128, o = tm + TM_O + i * 128;
                        auto part = [&](int x, int at, bool fresh) {         // 16 positions of the part in columns `at`
                            ta_mma_ts(o, p + 32 * (x >> 1) + at + 8 * (x & 1), v + x * (2048 >> 4), id_o, !fresh);
                        };
#pragma unroll
                        for (int x = 0; x < TA_KV / 16; ++x) {
                            part(x, 0, first && j == 0 && x == 0);
                            if constexpr (HILO && !THIRD) part(x, 16, false);
                        }
                        if (!last) {                                         // the third part comes while the product with the second runs
                            tc5_commit(h_used + 8 * i);
#pragma unroll
                            for (int x = 0; x < TA_KV / 16; ++x) part(x, 16, false);
                        } else if (j + 1 < e) {
                            scores(i, sk);
                        } else {
                            tc5_commit(o_full + 8 * i);
                        }
                    }
                    done[i]++;
                };
#pragma unroll
                for (int i = 0; i < TILES; ++i) {                    // a tile's parts follow one another, the other tile's softmax beside them
                    product(i, true, !THIRD);
                    if constexpr (THIRD) product(i, false, true);
                }
                if (ok && leader) {
                    tc5_commit(kv_empty + 8 * sv);
                    if (j + 1 < E) tc5_commit(kv_empty + 8 * sk);
                    if (j + 2 == E) tc5_commit(q_empty);
                }
            }
            it--;                                                    // the last round counted a K tile that was not there
            segs++;
            seg_done();
        }
        if (leader) tc5_commit(drain);                               // nothing of the tensor core's is left when TMEM is given back
        __syncwarp();
        if (!mbar_wait_ns(drain, 0, TA_DRAIN_NS)) *abort_flag = 1;
    } else if (warp == R::EDGES) {
        TA_REGS("dec", R::REGS_OTHER);
        // ------------------------------------------------ edges
        // V tiles at the edge of what the item's rows see. Positions behind the sequence's end become zeros (another sequence's rows,
        // or what was in the stage before), and so does what is infinite or NaN: its weight is zero for the rows that do not see it,
        // and 0 * inf is not. The rows that do see it get it back at the end (seg_odd).
        uint32_t it = 0, segs = 0, edges = 0;
        while (const volatile TaSeg *t = seg_next()) {
            const int u0 = t->u0, E = max(t->e[0], t->e[1]);
            if (E == 0) { seg_done(); continue; }
            const int edge = t->edge - u0, left = t->len - u0 * TA_KV;
            if (lane == 0) seg_odd[segs & 3] = 0;
            __syncwarp();
            for (int j = 0; j < E && ok; ++j, it += 2) {
                if (j < edge) continue;
                const uint32_t s = (it + 1) % L::STAGES;
                ok = __all_sync(0xffffffffu, ta_wait(e_full + 8 * (edges % L::OKS), (edges / L::OKS) & 1, abort_flag, true));
                if (!ok) break;
                const int rows = left - j * TA_KV;       // of the sequence
                const uint32_t v = sbase + L::KV + s * L::TILE;
                const int used = min(rows, TA_KV) * 8;               // 16-byte pieces of a half, eight to a row
                uint32_t seen = 0;
#pragma unroll
                for (int h = 0; h < L::NH; ++h) {
#pragma unroll 8
                    for (int x = lane; x < used; x += 32) {
                        uint32_t w[4];
                        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(v + h * L::HALF + x * 16));
                        // an exponent of all ones carries into the sign's place
#pragma unroll
                        for (int y = 0; y < 4; ++y) seen |= (w[y] & 0x7FFF7FFFu) + (BF16 ? 0x00800080u : 0x04000400u);
                    }
                    for (int x = used + lane; x < TA_KV * 8; x += 32)
                        asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(v + h * L::HALF + x * 16), "r"(0u) : "memory");
                }
                const bool odd = __any_sync(0xffffffffu, (seen & 0x80008000u) != 0);
                if (odd) {
#pragma unroll 1
                    for (int x = lane; x < L::NH * TA_KV * 8 * 4; x += 32) {
                        const uint32_t at = v + x * 4;
                        uint32_t w;
                        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(at));
                        const uint32_t f = ta_finite<BF16>(w);
                        if (f != w) asm volatile("st.shared.u32 [%0], %1;" ::"r"(at), "r"(f) : "memory");
                    }
                }
                if (odd) seg_odd[segs & 3] = 1;
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(v_ok + 8 * (edges % L::OKS));
                edges++;
            }
            segs++;
            seg_done();
        }
    } else if (warp == R::WALK) {
        TA_REGS("dec", R::REGS_OTHER);
        // ------------------------------------------------ the walk
        AttnCut first, last;
        attn_share(a, blockIdx.x, gridDim.x, TA_UNIT_SHIFT, min_units, first, last);
        AttnWalk walk;
        walk.begin(first, last);
        AttnSeg g;
        for (bool more = true; more && ok; ++gi) {
            if (gi >= TA_SEGS) ok = __all_sync(0xffffffffu, ta_wait(g_empty + 8 * (gi % TA_SEGS), (gi / TA_SEGS + 1) & 1, abort_flag, true));
            if (!ok) break;
            more = walk.next(a, TA_UNIT_SHIFT, g);
            if (lane == 0) {
                if (more) ta_seg<TILES>(a, g, ring + gi % TA_SEGS);
                else ring[gi % TA_SEGS].seq = -1;
                mbar_arrive(g_full + 8 * (gi % TA_SEGS));
            }
        }
    } else {
        TA_REGS("inc", R::REGS_SOFT);
        // ------------------------------------------------ softmax: warpgroup i owns tile i, a thread one of its rows
        // The weights of a tile are taken to a reference of the tiles before it, without looking for the tile's own maximum first (250
        // clocks): nothing is lost as long as they stay in range, and their sum, which is taken anyway, says whether they do. A row's
        // first reference is the largest of its first 16 scores (f16, whose weights have less room: of its first tile's). Where the sum
        // passes the limit (or is NaN), in masked tiles, and for f32 results, S is read for its maximum, O rescaled -- S's arrival tells
        // that the product before it is complete -- and the weights taken to that: S stays whole until P is written over it. The sums and
        // products are f32, so scaled by up to the limit they lose nothing. The two ways are kept apart: a loop around one of them, or
        // masks in it, cost 100 to 470 clocks a tile.
        const int i = warp >> 2, r = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;           // 32 lanes a warp, in bits 16 and up of a TMEM address
        const uint32_t S = tmem + i * 128 + lanes, O = tmem + TM_O + i * 128 + lanes;
        const float c = a.scale_log2;
        uint32_t tiles = 0, parts = 0, segs = 0;
        AttnMeta *const meta = a.meta + blockIdx.x;
        int flags = 0;                                               // of thread 0
        while (const volatile TaSeg *t = seg_next()) {
            const int E = t->e[i], p_first = t->u0 * TA_KV;
            const int tok = i * tq + r / a.g;                        // of the item
            const bool live = r < tq * a.g && tok < t->ntok;
            const int seen = ta_seen(t, t->tok0 + min(tok, t->ntok - 1) + 1) - p_first;      // positions of the segment that the row sees
            const int all_seen = ta_seen(t, t->tok0 + i * tq + 1) - p_first;                 // by the tile's first token: below it nothing is masked
            const bool idle = !__any_sync(0xffffffffu, live);        // no row of the warp is used: its columns of P stay as they are
            float m = -INFINITY, l = 0.f;                            // m: the reference that O and l are scaled to (of S, unscaled)
            for (int j = 0; j < E; ++j, ++tiles) {
                ok = __all_sync(0xffffffffu, ta_wait(s_full + 8 * i, tiles & 1, abort_flag));
                if (!ok) break;
                if (idle) {
                    if (lane == 0) mbar_arrive(p_full + 8 * i);
                    if constexpr (THIRD) {
                        ok = __all_sync(0xffffffffu, ta_wait(h_used + 8 * i, tiles & 1, abort_flag));
                        if (!ok) break;
                        if (lane == 0) mbar_arrive(p_full + 8 * i);
                    }
                    continue;
                }
                tc5_fence_after();
                const int n = seen - j * TA_KV;                      // positions of the tile that the row sees
                const bool masked = (j + 1) * TA_KV > all_seen;
                // 32 positions' weights, packed, (HILO) what the packing left, and (THIRD) what that one's left; their sum
                auto weights = [&](const uint32_t (&v)[32], float mc, float (&sum)[2][2], uint32_t (&hi)[16], uint32_t (&lo)[16], uint32_t (&th)[16]) {
#pragma unroll
                    for (int y = 0; y < 16; ++y) {
                        float u, w;
                        tc5_fma2(u, w, __uint_as_float(v[2 * y]), __uint_as_float(v[2 * y + 1]), c, mc);
                        u = ta_exp2(u);
                        w = ta_exp2(w);
                        if constexpr (!BF16 && HILO) { u *= 16384.f; w *= 16384.f; }       // 2^LOG_TOP, exact; else mc holds it
                        ta_add2(sum[y & 1], u, w);
                        hi[y] = ta_pack<BF16>(u, w);
                        if constexpr (HILO) {
                            const float2 b = ta_unpack<BF16>(hi[y]);
                            u -= b.x; w -= b.y;
                            lo[y] = ta_pack<BF16>(u, w);
                            if constexpr (THIRD) {
                                const float2 d = ta_unpack<BF16>(lo[y]);
                                th[y] = ta_pack<BF16>(u - d.x, w - d.y);
                            }
                        }
                    }
                };
                // what the scores' exponents start from
                auto minus = [&](float ref) { return ref == -INFINITY ? 0.f : BF16 || HILO ? -ref * c : fmaf(-ref, c, W::LOG_TOP); };
                bool slow = masked || HILO;
                if (BF16 && j == 0 && !slow) {                       // any of a row's scores may be the first reference
                    uint32_t v[16];
                    tc5_ld16(S, v);
                    ta_wait_ld(v);
                    float top[2] = {__uint_as_float(v[0]), __uint_as_float(v[1])};
#pragma unroll
                    for (int y = 2; y < 16; ++y) top[y & 1] = fmaxf(top[y & 1], __uint_as_float(v[y]));
                    m = fmaxf(top[0], top[1]);
                    if (!(m < INFINITY)) m = 0.f;                    // the sum tells of NaN and +inf
                }
                if (!slow) {
                    uint32_t s[4][32], hi[4][16], none[16];
                    float sum[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
                    for (int x = 0; x < 4; ++x) tc5_ld32(S + 32 * x, s[x]);
#pragma unroll
                    for (int x = 0; x < 4; ++x) ta_wait_ld(s[x]);
                    if (!BF16 && j == 0) {                           // f16 has less room over the reference: the largest of the tile
                        float top[4];
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            top[x] = __uint_as_float(s[x][0]);
#pragma unroll
                            for (int y = 1; y < 32; ++y) top[x] = fmaxf(top[x], __uint_as_float(s[x][y]));
                        }
                        m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                        if (!(m < INFINITY)) m = 0.f;
                    }
                    const float mc = minus(m);
#pragma unroll
                    for (int x = 0; x < 4; ++x) weights(s[x], mc, sum, hi[x], none, none);
                    const float total = (sum[0][0] + sum[1][0]) + (sum[0][1] + sum[1][1]);
                    slow = __any_sync(0xffffffffu, live && m == m && (!(total <= W::LIMIT) || (m == -INFINITY && total > 0.f)));
                    if (!slow) {
                        l += total;
#pragma unroll
                        for (int x = 0; x < 4; ++x) ta_st16(S + 32 * x, hi[x]);      // over the positions' own columns
                    }
                }
                uint32_t third[THIRD ? 4 : 1][16];
                if (slow) {
                    uint32_t s[4][32];
#pragma unroll
                    for (int x = 0; x < 4; ++x) tc5_ld32(S + 32 * x, s[x]);
#pragma unroll
                    for (int x = 0; x < 4; ++x) ta_wait_ld(s[x]);
                    if (!HILO || masked) {
#pragma unroll
                        for (int x = 0; x < 4; ++x)
#pragma unroll
                            for (int y = 0; y < 32; ++y)
                                if (32 * x + y >= n) s[x][y] = 0xFF800000u;
                    }
                    float tops[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        tops[x] = __uint_as_float(s[x][0]);
#pragma unroll
                        for (int y = 1; y < 32; ++y) tops[x] = ta_max(tops[x], __uint_as_float(s[x][y]));
                    }
                    const float top = ta_max(ta_max(tops[0], tops[1]), ta_max(tops[2], tops[3]));      // of the row; m, l and O go up to it,
                    // or (f32 results) stay where they are while the weights have room
                    const bool stay = HILO && !__any_sync(0xffffffffu, live && !((top - m) * c <= W::ROOM));
                    const float next = stay ? m : ta_max(m, top);    // NaN stays
                    const float f = next == m || next == -INFINITY ? 1.f : ta_exp2((m - next) * c);
                    m = next < INFINITY ? next : __int_as_float(0x7fffffff);      // a score of NaN or +inf: so is every weight of the row
                    l *= f;
                    if (j > 0 && __any_sync(0xffffffffu, f != 1.f)) {
#pragma unroll 1
                        for (int x = 0; x < D / 16; ++x) {
                            uint32_t o[16];
                            tc5_ld16(O + 16 * x, o);
                            ta_wait_ld(o);
#pragma unroll
                            for (int y = 0; y < 16; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * f);
                            ta_st16(O + 16 * x, o);
                        }
                    }
                    const float mc = minus(m);
                    float sum[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        uint32_t hi[16], lo[16];
                        weights(s[x], mc, sum, hi, lo, third[THIRD ? x : 0]);
                        ta_st16(S + 32 * x, hi);
                        if constexpr (HILO) ta_st16(S + 32 * x + 16, lo);
                    }
                    l += (sum[0][0] + sum[1][0]) + (sum[0][1] + sum[1][1]);
                }
                ta_wait_st();
                tc5_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + 8 * i);
                if constexpr (THIRD) {
                    ok = __all_sync(0xffffffffu, ta_wait(h_used + 8 * i, tiles & 1, abort_flag));
                    if (!ok) break;
                    tc5_fence_after();
#pragma unroll
                    for (int x = 0; x < 4; ++x) ta_st16(S + 32 * x, third[x]);
                    ta_wait_st();
                    tc5_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(p_full + 8 * i);
                }
            }
            if (!ok) break;
            const bool whole = t->whole;
            // sees nothing; or sees positions, and each of its scores is -inf
            if (m == -INFINITY) l = seen + p_first <= 0 ? 0.f : (whole ? __int_as_float(0x7fffffff) : ATTN_DARK);
            bool odd = false;
            if (E > 0) {
                ok = __all_sync(0xffffffffu, ta_wait(o_full + 8 * i, parts & 1, abort_flag));
                if (!ok) break;
                parts++;
                tc5_fence_after();
                if (seg_bad[segs & 3]) l = __int_as_float(0x7fffffff);
                odd = seg_odd[segs & 3];
            }
            const int row = i * tq * a.g + r;                        // of the item
            float *slot = nullptr;
            if (!whole) {
                const int which = t->u0 > 0 ? 0 : 1;
                slot = a.part + ((size_t)blockIdx.x * 2 + which) * attn_slot_floats(R::ROWS, D);
                if (threadIdx.x == 0) {
                    if (which == 0) flags |= ATTN_CONT | (t->ends ? ATTN_ENDS : 0);
                    else { flags |= ATTN_OWN; meta->row = t->row + t->tok0; meta->ntok = t->ntok; meta->head = t->head; }
                }
                if (live) {
                    slot[R::ROWS * D + row] = m * c;
                    slot[R::ROWS * D + R::ROWS + row] = l;
                }
            }
            const float inv = whole ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
            // Rows leave through shared memory, PASS bytes of each at a time: a thread has a row, and its own stores would touch 32 lines
            // an instruction (8 us of an item's time). Where the row goes; negative: nowhere.
            constexpr int PB = L::PASS, GR = PB / 4, PP = PB / 16;   // columns fetched at a time; 16-byte pieces of a row's pass
            const bool f32 = !whole || a.out_dtype == JL_DT_F32;
            const int size = f32 ? 4 : 2;
            uint8_t *const dst = whole ? static_cast<uint8_t *>(a.out) + ((long long)(t->row + t->tok0) * a.hq + t->head * a.g) * size * D
                                       : reinterpret_cast<uint8_t *>(slot);      // of the item
            const int at = !live || (!whole && E == 0) ? -1 : (whole ? tok * a.hq + r % a.g : row) * size * D;
            const uint32_t stage = sbase + L::OUT + warp * 32 * PB;
            auto swizzle = [](int row, int piece) { return PP == 8 ? piece ^ (row & 7) : piece ^ ((row >> 1) & 3); };
            const int first = lane / PP, pc = lane % PP;             // of the rows and pieces that this thread stores: rows first + y 32 / PP
            int to[PP];
#pragma unroll
            for (int y = 0; y < PP; ++y) to[y] = __shfl_sync(0xffffffffu, at, y * (32 / PP) + first);
            uint32_t w[GR];                                          // the pass
#pragma unroll 1
            for (int x = 0; x < D / GR && !idle; ++x) {
                uint32_t o[GR];
                if (E > 0) {
                    if constexpr (GR == 32) tc5_ld32(O + GR * x, o);
                    else tc5_ld16(O + GR * x, o);
                    ta_wait_ld(o);
                } else {
#pragma unroll
                    for (int y = 0; y < GR; ++y) o[y] = 0u;
                }
                if (f32) {
#pragma unroll
                    for (int y = 0; y < GR; ++y) w[y] = __float_as_uint(__uint_as_float(o[y]) * inv);
                } else {
#pragma unroll
                    for (int y = 0; y < GR / 2; ++y) {
                        const float u = __uint_as_float(o[2 * y]) * inv, v = __uint_as_float(o[2 * y + 1]) * inv;
                        const uint32_t p = a.out_dtype == JL_DT_BF16 ? ta_pack<true>(u, v) : ta_pack<false>(u, v);
                        if (x & 1) w[GR / 2 + y] = p; else w[y] = p;
                    }
                    if (!(x & 1)) continue;
                }
                __syncwarp();                                        // the last pass's rows have been read
#pragma unroll
                for (int y = 0; y < PP; ++y)
                    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(stage + lane * PB + (swizzle(lane, y) << 4)), "r"(w[4 * y]),
                                 "r"(w[4 * y + 1]), "r"(w[4 * y + 2]), "r"(w[4 * y + 3]) : "memory");
                __syncwarp();
                const int col = f32 ? PB * x : PB / 2 * (x - 1);     // in bytes
#pragma unroll
                for (int y = 0; y < PP; ++y) {
                    const int rr = y * (32 / PP) + first;
                    uint4 v;
                    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                                 : "r"(stage + rr * PB + (swizzle(rr, pc) << 4)));
                    if (to[y] >= 0) *reinterpret_cast<uint4 *>(dst + to[y] + col + 16 * pc) = v;
                }
            }
            __syncwarp();
            if (odd && at >= 0)
                ta_odd<BF16>(&a, t->seq, t->head, t->row, max(t->u0, t->edge) * TA_KV, p_first + min(seen, E * TA_KV), dst + at, f32 ? JL_DT_F32 : a.out_dtype);
            if (max(t->e[0], t->e[1]) > 0) segs++;
            seg_done();
        }
        if (threadIdx.x == 0) meta->flags = flags;
    }
    tc5_fence_before();
    __syncthreads();
    tc5_fence_after();
    if (threadIdx.x == 0 && *abort_flag) atomicExch(a.status, TA_STATUS_CODE);
    if (warp == R::MMA) tc5_dealloc(tmem, 256 * TILES);
}

static bool ta_map(CUtensorMap *map, const void *base, bool bf16, int rank, const cuuint64_t *dims, const cuuint64_t *strides, const cuuint32_t *box) {
    jl_encode_tiled_fn enc = jl_get_encode_tiled();
    if (!enc) return false;
    const cuuint32_t one[4] = {1, 1, 1, 1};
    return enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, const_cast<void *>(base), dims, strides, box, one,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int TILES, bool BF16, bool HILO>
static int ta_go(jl_ctx *ctx, const AttnArgs &a, const CUtensorMap &q, const CUtensorMap &k, const CUtensorMap &v, int box_rows, cudaStream_t s) {
    using R = TaRoles<TILES>;
    auto kern = attn_tc5_kernel<D, TILES, BF16, HILO>;
    const int smem = TaSmem<D, TILES>::TOTAL, grid = ctx->sm_count * R::CTAS;
    JL_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    const cudaError_t e = attn_launch_pdl(ctx, kern, dim3(grid), dim3(R::WARPS * 32), smem, s, a, q, k, v, box_rows, 2);
    JL_CUDA(ctx, e);
    ctx->st.launches++;
    return attn_launch_merge(ctx, a, R::ROWS, grid, TA_KV, s);
}

template <int D, int TILES>
static int ta_type(jl_ctx *ctx, const AttnArgs &a, bool bf16, const CUtensorMap &q, const CUtensorMap &k, const CUtensorMap &v, int box_rows, cudaStream_t s) {
    if (a.out_dtype == JL_DT_F32)
        return bf16 ? ta_go<D, TILES, true, true>(ctx, a, q, k, v, box_rows, s) : ta_go<D, TILES, false, true>(ctx, a, q, k, v, box_rows, s);
    return bf16 ? ta_go<D, TILES, true, false>(ctx, a, q, k, v, box_rows, s) : ta_go<D, TILES, false, false>(ctx, a, q, k, v, box_rows, s);
}

int attn_launch_tc5(jl_ctx *ctx, const AttnArgs &args, int dtype, long long max_rows, cudaStream_t s) {
    AttnArgs a = args;
    const int tq = 128 / a.g, tiles = max_rows <= TA_ONE_TILE_ROWS ? 1 : 2;
    a.tok_item = tiles * tq;
    a.item_cost = tiles == 1 ? TA_ITEM_COST_ONE : TA_ITEM_COST;
    a.snap = tiles == 1 ? 0 : TA_SNAP;
    const bool bf16 = dtype == JL_DT_BF16;
    CUtensorMap q, k, v;
    const cuuint64_t d = a.d;
    const cuuint64_t qd[3] = {d, (cuuint64_t)a.hq, (cuuint64_t)a.total}, qs[2] = {(cuuint64_t)a.q_head * 2, (cuuint64_t)a.q_tok * 2};
    const cuuint32_t qb[3] = {64, (cuuint32_t)a.g, (cuuint32_t)tq};
    const int box_rows = a.table ? (a.page_shift < TA_UNIT_SHIFT ? 1 << a.page_shift : TA_KV) : TA_KV;
    const cuuint64_t rows = a.table ? (cuuint64_t)1 << a.page_shift : (cuuint64_t)a.total, pages = a.table ? (cuuint64_t)a.n_pages : 1;
    const cuuint64_t kd[4] = {d, rows, (cuuint64_t)a.hkv, pages};
    const cuuint64_t ks[3] = {(cuuint64_t)a.kv_tok * 2, (cuuint64_t)a.kv_head * 2, a.table ? (cuuint64_t)a.kv_page * 2 : (cuuint64_t)a.kv_tok * 2};
    const cuuint32_t kb[4] = {64, (cuuint32_t)box_rows, 1, 1};
    if (!ta_map(&q, a.q, bf16, 3, qd, qs, qb) || !ta_map(&k, a.k, bf16, 4, kd, ks, kb) || !ta_map(&v, a.v, bf16, 4, kd, ks, kb))
        return jl_set_err(ctx, JL_ENOTSUP, "attention: the driver makes no tensor map of these strides");       // it does of all that are let through
    if (tiles == 1) return a.d == 128 ? ta_type<128, 1>(ctx, a, bf16, q, k, v, box_rows, s) : ta_type<64, 1>(ctx, a, bf16, q, k, v, box_rows, s);
    return a.d == 128 ? ta_type<128, 2>(ctx, a, bf16, q, k, v, box_rows, s) : ta_type<64, 2>(ctx, a, bf16, q, k, v, box_rows, s);
}
