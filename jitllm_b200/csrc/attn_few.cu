// Attention for few query rows: the new tokens of a sequence times the query heads of a kv head are taken sixteen rows at a time,
// the height of one mma.sync tile, so that the keys and values of a position are read once for all of them.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(scale log2(e) q.k_j - m),  m the largest exponent so far
//
// Per position and kv head 4 d bytes are read for 48 d multiply-adds (64 d for f32 results of bf16): bound by the cache's bytes. A CTA is
// four warps; a unit is 64 positions, 16 of them a warp's, and each warp runs its own cp.async ring, running maximum, sum and accumulators:
// no warp waits for another before the end of the CTA's positions. mma.sync, not tcgen05: the products are a few percent of the tensor
// cores' time, and an accumulator in registers needs no barrier between a tile's softmax and its product with V.
//
// Measured: 64 sequences of 37 to 8200 positions, 32 heads over 8, 408 MB: 89 us, 4.6 TB/s. The loop itself reads at 6.0 TB/s (long
// sequences of equal length, 1.3 GB: 5.4 TB/s with everything); the rest is the share's start (4 us: lengths, table, first tiles, one after the
// other), items' starts and ends, the last CTAs' 8 us and the join (6 us). Few positions are latency: 2049 of one sequence take 16 us.
// Tried and not kept: a ring that runs on into the next item while this one's sums are joined, 16 columns at a time (the join of the warps
// costs what the loads save, the other CTAs of the SM fill the gap anyway: a microsecond slower).
#include "attn.cuh"

#define FEW_UNIT_SHIFT 6
#define FEW_STAGES 2
// In units, for 64 sequences of 37 to 8200 positions:
#define FEW_ITEM_COST 4          // an item's start and end: 1, 2, 3 and 4 take 105, 96, 89 and 89 us
#define FEW_SNAP 2               // 0, 2 and 6 take 90, 89 and 96 us
#define FEW_MIN_UNITS 2          // of a share: 1 and 2 take 16.2 and 16.0 us for 2049 positions: twice the parts to join

template <int D> struct FewTile {
    static constexpr int ROW = 2 * D + 16;            // bytes of a staged row: padded, so that rows start in different banks
    static constexpr int BYTES = 2 * 16 * ROW;        // 16 rows of K, 16 of V
    static constexpr int SMEM = 4 * FEW_STAGES * BYTES;
};

__device__ __forceinline__ float few_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <bool BF16>
__device__ __forceinline__ void few_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The largest weight so far. f16 ends at 2^-24, so its weights are taken to 2^14 instead of one: a weight is then held to 2^-39 of the
// largest, where a long flat tail below 2^-25 of it would leave the products but not the sum (131,071 positions: 0.4 % of a result).
template <bool BF16> __device__ constexpr float few_top() { return BF16 ? 1.f : 16384.f; }
// Two softmax weights in 16 bits, and what that rounding left of them.
template <bool BF16>
__device__ __forceinline__ uint32_t few_pack(float x, float y, float &rx, float &ry) {
    if constexpr (BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        const float2 b = __bfloat1622float2(h);
        rx = x - b.x; ry = y - b.y;
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __half2 h = __floats2half2_rn(x, y);
        const float2 b = __half22float2(h);
        rx = x - b.x; ry = y - b.y;
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}
template <bool BF16>
__device__ __forceinline__ float2 few_unpack(uint32_t w) {
    if constexpr (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    else return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
// Is either of two packed values infinite or NaN?
template <bool BF16>
__device__ __forceinline__ bool few_odd(uint32_t w) {
    constexpr uint32_t E = BF16 ? 0x7F80u : 0x7C00u;
    return (w & E) == E || (w & (E << 16)) == (E << 16);
}

template <int D, bool BF16, bool THIRD>
__global__ void __launch_bounds__(128, 3) attn_few_kernel(const __grid_constant__ AttnArgs a, int min_units) {
    constexpr int ROW = FewTile<D>::ROW, TILE = FewTile<D>::BYTES, NJ = D / 8, CH = D / 8;   // CH: 16-byte pieces of a row
    extern __shared__ __align__(16) uint8_t tiles[];   // the warps' rings; the cross-warp sum red[4][16][D] reuses them
    static_assert(4 * 16 * D * 4 <= FewTile<D>::SMEM, "the reduction fits in the rings");
    __shared__ float mred[4][16], lred[4][16];
    __shared__ int bad;
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31, gid = lane >> 2, tq = lane & 3;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    AttnCut first, last;
    attn_share(a, blockIdx.x, gridDim.x, FEW_UNIT_SHIFT, min_units, first, last);
    AttnMeta meta = {0, 0, 0, 0};
    AttnWalk walk;
    walk.begin(first, last);
    AttnSeg sg, ng;
    if (t == 0) bad = 0;
    const uint16_t *kp = static_cast<const uint16_t *>(a.k), *vp = static_cast<const uint16_t *>(a.v);
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(tiles) + warp * FEW_STAGES * TILE;
    // the page of the warp's tile i: 16 positions lie in one (pages are 16 positions at least, cut at multiples of their length)
    auto page_of = [&](const AttnSeg &g, int i) -> int {
        const int p = (g.u0 + i) * 64 + warp * 16;
        if (!a.table || i >= g.u1 - g.u0 || p >= g.q.len) return 0;
        return a.table[(long long)g.seq * a.max_pages + (p >> a.page_shift)];
    };
    bool more = walk.next(a, FEW_UNIT_SHIFT, ng);
    int page0 = more ? page_of(ng, 0) : 0, page1 = more ? page_of(ng, 1) : 0;
    while (more) {
        sg = ng;
        __syncthreads();                               // bad is set; the last segment's sums are read
        const int tok0 = sg.blk * a.tok_item, ntok = min(a.tok_item, sg.q.n - tok0);
        const int ntile = sg.u1 - sg.u0, base = sg.u0 * 64 + warp * 16;
        auto issue = [&](int i, int page) {
            if (i >= ntile) return;
            const int p = base + i * 64;
            const uint32_t dst = ring + (i % FEW_STAGES) * TILE;
            int rows = min(16, sg.q.len - p);          // rows past the sequence arrive as zeros
            long long at;
            if (a.table) {
                if (rows > 0 && (unsigned)page >= (unsigned)a.n_pages) { rows = 0; bad = 1; }
                if (rows <= 0) page = 0;
                at = page * a.kv_page + sg.head * a.kv_head + (p & ((1 << a.page_shift) - 1)) * a.kv_tok;
            } else {
                at = (long long)(sg.q.row + (rows > 0 ? p : 0)) * a.kv_tok + sg.head * a.kv_head;
            }
#pragma unroll
            for (int j = 0; j < CH / 2; ++j) {
                const int piece = j * 32 + lane, r = piece / CH, c = piece % CH, bytes = r < rows ? 16 : 0;
                const long long o = at + (r < rows ? r : 0) * a.kv_tok + c * 8;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + r * ROW + c * 16), "l"(kp + o), "r"(bytes) : "memory");
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + (16 + r) * ROW + c * 16), "l"(vp + o), "r"(bytes) : "memory");
            }
        };
        // Two tiles on their way before anything else is looked up; what the next segment needs is asked for while they come.
        issue(0, page0);
        asm volatile("cp.async.commit_group;" ::: "memory");
        issue(1, page1);
        asm volatile("cp.async.commit_group;" ::: "memory");
        int page = page_of(sg, 2);
        // rows of this thread: gid and gid + 8; row r is token tok0 + r / g, query head r % g of the kv head
        int seen[2];                                   // positions that the row sees
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = gid + 8 * e, tk = r / a.g;
            seen[e] = tk < ntok ? attn_limit(sg.q, tok0 + tk + 1) : 0;
        }
        const int few_seen = attn_limit(sg.q, tok0 + 1);            // of the item's first token: below it every row sees everything
        // q (and the table) by plain loads: the kernel in front, which may still have run when this one was put in place, can have written
        // it, and the read-only path is for what nothing writes while the kernel is there
        uint32_t qa[D / 16][4];
        {
            const uint16_t *qp = static_cast<const uint16_t *>(a.q);
            const uint32_t *row[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = gid + 8 * e, tk = min(r / a.g, ntok - 1);
                row[e] = reinterpret_cast<const uint32_t *>(qp + (long long)(sg.q.row + tok0 + tk) * a.q_tok +
                                                            (long long)(sg.head * a.g + r % a.g) * a.q_head);
            }
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
                qa[ks][0] = row[0][ks * 8 + tq]; qa[ks][1] = row[1][ks * 8 + tq];
                qa[ks][2] = row[0][ks * 8 + 4 + tq]; qa[ks][3] = row[1][ks * 8 + 4 + tq];
            }
        }
        more = walk.next(a, FEW_UNIT_SHIFT, ng);
        if (more) { page0 = page_of(ng, 0); page1 = page_of(ng, 1); }
        float M[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};     // of rows gid, gid + 8 (l: this lane's share)
        float oacc[NJ][4];                                          // O[gid][8 j + 2 tq, + 1], O[gid + 8][same]
#pragma unroll
        for (int j = 0; j < NJ; ++j) oacc[j][0] = oacc[j][1] = oacc[j][2] = oacc[j][3] = 0.f;
#pragma unroll 1
        for (int i = 0; i < ntile; ++i) {
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            __syncwarp();
            const uint32_t tile = ring + (i % FEW_STAGES) * TILE;
            const int p = base + i * 64;
            // S[row][pos]: two n-tiles of 8 positions; sv[nt][2 e + x] = S[gid + 8 e][p + 8 nt + 2 tq + x]
            float sv[2][4];
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
#pragma unroll
                for (int x = 0; x < 4; ++x) sv[nt][x] = 0.f;
#pragma unroll
                for (int kp2 = 0; kp2 < D / 32; ++kp2) {            // two k-steps (32 dims) per ldmatrix.x4
                    const uint32_t addr = tile + (8 * nt + (lane & 7)) * ROW + (32 * kp2 + 8 * (lane >> 3)) * 2;
                    uint32_t b0, b1, b2, b3;
                    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                                 : "=r"(b0), "=r"(b1), "=r"(b2), "=r"(b3) : "r"(addr));
                    few_mma<BF16>(sv[nt], qa[2 * kp2], b0, b1);
                    few_mma<BF16>(sv[nt], qa[2 * kp2 + 1], b2, b3);
                }
            }
            float keep[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float m = -INFINITY;
#pragma unroll
                for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        float &s = sv[nt][2 * e + x];
                        s = p + 8 * nt + 2 * tq + x < seen[e] ? s * a.scale_log2 : -INFINITY;
                        m = fmaxf(m, s);
                    }
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                m = fmaxf(m, M[e]);
                const float mu = m == -INFINITY ? 0.f : m;          // nothing seen yet: every weight is 2^-inf
                keep[e] = few_exp2(M[e] - mu);
                M[e] = m;
                l[e] *= keep[e];
#pragma unroll
                for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        float &s = sv[nt][2 * e + x];
                        s = few_exp2(s - mu) * few_top<BF16>();     // exact: a power of two
                        l[e] += s;
                    }
            }
            // A fragments of the weights, as value + remainder (16 significant bits of bf16, 22 of f16), and for f32 results of bf16
            // the remainder's remainder (24): the products with V lose nothing that the result shows. (An instance of its own: for 16-bit
            // results the third part would cost 0.8 of 88 us, 64 sequences.)
            uint32_t ph[4], pl[4], pt[4];
#pragma unroll
            for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float rx, ry, z0, z1;
                    ph[2 * nt + e] = few_pack<BF16>(sv[nt][2 * e], sv[nt][2 * e + 1], rx, ry);
                    pl[2 * nt + e] = few_pack<BF16>(rx, ry, z0, z1);
                    if constexpr (THIRD) { float y0, y1; pt[2 * nt + e] = few_pack<BF16>(z0, z1, y0, y1); }
                }
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                oacc[j][0] *= keep[0]; oacc[j][1] *= keep[0]; oacc[j][2] *= keep[1]; oacc[j][3] *= keep[1];
            }
            // Where some rows of the tile see a position and others do not, an infinite or NaN value there would reach the others
            // as 0 * inf: such a tile (of a sequence's own later tokens) is summed without the matrix instructions.
            bool odd = false;
            const bool edge = p + 15 >= few_seen;
            if (edge) {
                for (int x = lane; x < 16 * CH; x += 32) {
                    uint32_t w[4];
                    const uint32_t addr = tile + (16 + x / CH) * ROW + (x % CH) * 16;
                    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
#pragma unroll
                    for (int y = 0; y < 4; ++y) odd = odd || few_odd<BF16>(w[y]);
                }
                odd = __any_sync(0xffffffffu, odd);
            }
            if (!odd) {
#pragma unroll
                for (int jp = 0; jp < D / 16; ++jp) {
                    // matrices: V[0..7][dims 16 jp + 0..7], V[8..15][same], V[0..7][dims 16 jp + 8..15], V[8..15][same]
                    const int mi = lane >> 3;
                    const uint32_t addr = tile + (16 + 8 * (mi & 1) + (lane & 7)) * ROW + (16 * jp + 8 * (mi >> 1)) * 2;
                    uint32_t b0, b1, b2, b3;
                    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                                 : "=r"(b0), "=r"(b1), "=r"(b2), "=r"(b3) : "r"(addr));
                    few_mma<BF16>(oacc[2 * jp], ph, b0, b1);
                    few_mma<BF16>(oacc[2 * jp], pl, b0, b1);
                    few_mma<BF16>(oacc[2 * jp + 1], ph, b2, b3);
                    few_mma<BF16>(oacc[2 * jp + 1], pl, b2, b3);
                    if constexpr (THIRD) {
                        few_mma<BF16>(oacc[2 * jp], pt, b0, b1);
                        few_mma<BF16>(oacc[2 * jp + 1], pt, b2, b3);
                    }
                }
            } else {
#pragma unroll 1
                for (int x = 0; x < 16; ++x) {
                    const int nt = x >> 3, src = (lane & ~3) | ((x & 7) >> 1);
                    float w[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float even = nt ? sv[1][2 * e] : sv[0][2 * e], uneven = nt ? sv[1][2 * e + 1] : sv[0][2 * e + 1];
                        w[e] = __shfl_sync(0xffffffffu, x & 1 ? uneven : even, src);
                    }
#pragma unroll
                    for (int j = 0; j < NJ; ++j) {
                        uint32_t v;
                        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(tile + (16 + x) * ROW + (8 * j + 2 * tq) * 2));
                        const float2 f = few_unpack<BF16>(v);
                        if (p + x < seen[0]) { oacc[j][0] = fmaf(w[0], f.x, oacc[j][0]); oacc[j][1] = fmaf(w[0], f.y, oacc[j][1]); }
                        if (p + x < seen[1]) { oacc[j][2] = fmaf(w[1], f.x, oacc[j][2]); oacc[j][3] = fmaf(w[1], f.y, oacc[j][3]); }
                    }
                }
            }
            __syncwarp();                                           // every lane is done with the stage that is refilled now
            issue(i + 2, page);
            asm volatile("cp.async.commit_group;" ::: "memory");
            page = page_of(sg, i + 3);
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
            if (tq == 0) { mred[warp][gid + 8 * e] = M[e]; lred[warp][gid + 8 * e] = l[e]; }
        }
        __syncthreads();                                            // every warp's tiles are consumed: reuse them
        float(*red)[16][D] = reinterpret_cast<float(*)[16][D]>(tiles);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = gid + 8 * e;
            const float m = fmaxf(fmaxf(mred[0][r], mred[1][r]), fmaxf(mred[2][r], mred[3][r]));
            const float f = few_exp2(M[e] - (m == -INFINITY ? 0.f : m));
#pragma unroll
            for (int j = 0; j < NJ; ++j)
                *reinterpret_cast<float2 *>(&red[warp][r][8 * j + 2 * tq]) = make_float2(oacc[j][2 * e] * f, oacc[j][2 * e + 1] * f);
        }
        __syncthreads();
        const bool whole = sg.u0 == 0 && sg.u1 == sg.units;
        float *slot = nullptr;
        if (!whole) {
            const int which = sg.u0 > 0 ? 0 : 1;
            slot = a.part + ((size_t)blockIdx.x * 2 + which) * attn_slot_floats(ATTN_FEW_ROWS, D);
            if (which == 0) meta.flags |= ATTN_CONT | (sg.u1 == sg.units ? ATTN_ENDS : 0);
            else { meta.flags |= ATTN_OWN; meta.row = sg.q.row + tok0; meta.ntok = ntok; meta.head = sg.head; }
        }
        for (int x = t; x < 16 * (D / 4); x += 128) {
            const int r = x / (D / 4), c = x % (D / 4);
            const float m = fmaxf(fmaxf(mred[0][r], mred[1][r]), fmaxf(mred[2][r], mred[3][r])), mu = m == -INFINITY ? 0.f : m;
            float L = 0.f;
            float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                L += lred[w][r] * few_exp2(mred[w][r] - mu);
                const float4 v = *reinterpret_cast<const float4 *>(&red[w][r][4 * c]);
                s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
            }
            const int tk = r / a.g;
            if (L == 0.f && tk < ntok && attn_limit(sg.q, tok0 + tk + 1) > 0)       // sees positions, and each of its scores is -inf
                L = whole ? __int_as_float(0x7fffffff) : ATTN_DARK;
            if (bad || sg.q.over) L = __int_as_float(0x7fffffff);   // a page outside the pool, positions outside the table: NaN
            if (whole) {
                if (tk < ntok) {
                    const float inv = L == 0.f ? 0.f : 1.f / L;     // a row that sees nothing is zero
                    if (L == 0.f) s = make_float4(0.f, 0.f, 0.f, 0.f);
                    attn_store4(a.out, a.out_dtype, ((size_t)(sg.q.row + tok0 + tk) * a.hq + sg.head * a.g + r % a.g) * D + 4 * c,
                                make_float4(s.x * inv, s.y * inv, s.z * inv, s.w * inv));
                }
            } else {
                *reinterpret_cast<float4 *>(slot + (size_t)r * D + 4 * c) = s;
                if (c == 0) { slot[16 * D + r] = m; slot[16 * D + 16 + r] = L; }
            }
        }
        __syncthreads();
        if (t == 0) bad = 0;
    }
    if (t == 0) a.meta[blockIdx.x] = meta;
}

template <int D, bool BF16, bool THIRD>
static int few_go(jl_ctx *ctx, const AttnArgs &a, cudaStream_t s) {
    const int smem = FewTile<D>::SMEM, grid = attn_few_grid(ctx);
    auto kern = attn_few_kernel<D, BF16, THIRD>;
    if (smem > 48 * 1024) JL_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    const cudaError_t e = attn_launch_pdl(ctx, kern, dim3(grid), dim3(128), smem, s, a, FEW_MIN_UNITS);
    JL_CUDA(ctx, e);
    ctx->st.launches++;
    return attn_launch_merge(ctx, a, ATTN_FEW_ROWS, grid, 1 << FEW_UNIT_SHIFT, s);
}

int attn_launch_few(jl_ctx *ctx, const AttnArgs &args, int dtype, cudaStream_t s) {
    AttnArgs a = args;
    a.tok_item = ATTN_FEW_ROWS / a.g;
    a.item_cost = FEW_ITEM_COST;
    a.snap = FEW_SNAP;
    const bool third = a.out_dtype == JL_DT_F32;
    if (dtype != JL_DT_BF16) return a.d == 128 ? few_go<128, false, false>(ctx, a, s) : few_go<64, false, false>(ctx, a, s);
    if (a.d == 128) return third ? few_go<128, true, true>(ctx, a, s) : few_go<128, true, false>(ctx, a, s);
    return third ? few_go<64, true, true>(ctx, a, s) : few_go<64, true, false>(ctx, a, s);
}
