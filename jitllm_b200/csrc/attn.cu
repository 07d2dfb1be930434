// Several sequences at once: attention over packed prompts, attention of new tokens over a cache in pages, and the cache's writer.
// The entry points, the join of partial results and the writer; the attention kernels are in attn_few.cu and attn_tc5.cu.
#include "attn.cuh"

#include <limits.h>
#include <math.h>

// ------------------------------------------------------------------ join of partial results
// The item that CTA c began, and the CTAs behind it continued: the softmax weights of the parts are 2^(their maximum - the largest), the
// parts added in ascending order of positions.

// What a warp knows of it after one round of loads: meta of CTA c + lane, and the item's parts, c to c + n - 1 (a CTA among them whose
// share came out empty has none).
struct AttnItem { int flags, row, ntok, head, n; };
__device__ __forceinline__ AttnItem attn_item(const AttnMeta *meta, int c, int ctas) {
    const int lane = threadIdx.x & 31;
    const int4 m = *reinterpret_cast<const int4 *>(meta + min(c + lane, ctas - 1));
    AttnItem it;
    it.flags = lane == 0 || (m.x & ATTN_CONT);                    // does CTA c + lane hold a part?
    it.row = __shfl_sync(0xffffffffu, m.y, 0); it.ntok = __shfl_sync(0xffffffffu, m.z, 0); it.head = __shfl_sync(0xffffffffu, m.w, 0);
    it.n = 0;
    if (!(__shfl_sync(0xffffffffu, m.x, 0) & ATTN_OWN)) return it;
    unsigned b = __ballot_sync(0xffffffffu, lane > 0 && (c + lane >= ctas - 1 || (m.x & ATTN_ENDS)));
    int at = c;
    while (!b) {                                                  // eight of a lane's looks on their way at a time
        unsigned e[8];
        at += 32;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int i = min(at + 32 * k + lane, ctas - 1);
            e[k] = i == ctas - 1 || (meta[i].flags & ATTN_ENDS);
        }
        int to = at;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const unsigned x = __ballot_sync(0xffffffffu, e[k]);
            if (x && !b) { b = x; to = at + 32 * k; }
        }
        at = b ? to : at + 224;
    }
    it.n = min(at + __ffs(b) - 1, ctas - 1) - c + 1;
    return it;
}
template <int D>
__device__ __forceinline__ void attn_merge_store(const AttnArgs &a, const AttnItem &own, int r, int col, const float (&acc)[D / 32], float L) {
    const float inv = L == 0.f ? 0.f : 1.f / L;
    const size_t at = ((size_t)(own.row + r / a.g) * a.hq + own.head * a.g + r % a.g) * D + col;
    if constexpr (D == 128) attn_store4(a.out, a.out_dtype, at, make_float4(acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv));
    else attn_store2(a.out, a.out_dtype, at, acc[0] * inv, acc[1] * inv);
}
template <int D>
__device__ __forceinline__ void attn_merge_load(const float *p, float (&v)[D / 32]) {
    if constexpr (D == 128) {
        const float4 u = __ldcg(reinterpret_cast<const float4 *>(p));
        v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
    } else {
        const float2 u = __ldcg(reinterpret_cast<const float2 *>(p));
        v[0] = u.x; v[1] = u.y;
    }
}

// Bound by the latency of loads that follow one another, 0.7 us each beside parts of a few MB that L2 serves: so everything whose address
// is known is asked for at once, the maxima, the sums and the first parts' rows, and weighed once it is there.

// Many rows and, as a rule, few parts: block (c, y) takes 16 rows, a warp two of them side by side. One row to a warp needs four waves of
// blocks (five tokens of 32 sequences 50 us in all, 24 prompts 61.7; with two rows 48.5 and 60.8), four take registers from the loads'
// overlap (50, 61.4, 1531 tokens 52.7 instead of 50.5; a mixed step 142 instead of 138). Four of the parts' rows ahead instead of two: 1531 tokens
// 52.4, the step 140.
#define ATTN_MERGE_ROWS 2
#define ATTN_MERGE_AHEAD 2
template <int D>
__global__ void __launch_bounds__(256) attn_merge_many_kernel(const __grid_constant__ AttnArgs a, int ctas, int slot_rows) {
    constexpr int V = D / 32, B = ATTN_MERGE_AHEAD, R = ATTN_MERGE_ROWS;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int c = blockIdx.x, lane = threadIdx.x & 31, r0 = (blockIdx.y * 8 + (threadIdx.x >> 5)) * R;
    const AttnItem it = attn_item(a.meta, c, ctas);
    const int rows = min(R, it.ntok * a.g - r0);
    if (!it.n || rows <= 0) return;
    const size_t slot = attn_slot_floats(slot_rows, D);
    auto part_of = [&](int k) { return a.part + ((size_t)(c + k) * 2 + (k == 0)) * slot; };
    auto there = [&](int k) { return k < it.n && (k < 32 ? it.flags : a.meta[c + k].flags & ATTN_CONT) != 0; };      // k % 32 == lane
    float v[R][B][V], m[R], l[R], M[R], L[R], acc[R][V];
    bool dark[R];
    auto heads_of = [&](int k) {                                     // the rows' maxima and sums in part k
        const bool has = there(k);
        const float *p = part_of(k) + slot_rows * D + r0;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            m[i] = has && i < rows ? __ldcg(p + i) : -INFINITY;
            l[i] = has && i < rows ? __ldcg(p + slot_rows + i) : 0.f;
        }
    };
    auto rows_of = [&](int k0) {
#pragma unroll
        for (int k = 0; k < B; ++k)
#pragma unroll
            for (int i = 0; i < R; ++i)
                if (k0 + k < it.n && i < rows) attn_merge_load<D>(part_of(k0 + k) + (size_t)(r0 + i) * D + V * lane, v[i][k]);
    };
    heads_of(lane);
    rows_of(0);
#pragma unroll
    for (int i = 0; i < R; ++i) {
        M[i] = m[i];
        L[i] = 0.f;
        dark[i] = __shfl_sync(0xffffffffu, l[i], 0) < 0.f;           // said by the first part, which every row that sees anything sees
#pragma unroll
        for (int x = 0; x < V; ++x) acc[i][x] = 0.f;
    }
    for (int k = 32 + lane; k < it.n; k += 32)
        if (there(k)) {
#pragma unroll
            for (int i = 0; i < R; ++i)
                if (i < rows) M[i] = fmaxf(M[i], __ldcg(part_of(k) + slot_rows * D + r0 + i));
        }
#pragma unroll
    for (int i = 0; i < R; ++i) {
#pragma unroll
        for (int o = 16; o; o >>= 1) M[i] = fmaxf(M[i], __shfl_xor_sync(0xffffffffu, M[i], o));
        M[i] = M[i] == -INFINITY ? 0.f : M[i];
    }
    for (int k0 = 0; k0 < it.n; k0 += B) {
        if (k0 && !(k0 & 31)) heads_of(k0 + lane);
        if (k0) rows_of(k0);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const float w = exp2f(m[i] - M[i]);
#pragma unroll
            for (int k = 0; k < B; ++k) {
                const float wk = __shfl_sync(0xffffffffu, w, (k0 + k) & 31), lk = __shfl_sync(0xffffffffu, l[i], (k0 + k) & 31);
                if (k0 + k >= it.n || lk <= 0.f) continue;        // the part holds nothing of this row, perhaps not even numbers
                L[i] = fmaf(wk, lk, L[i]);
#pragma unroll
                for (int x = 0; x < V; ++x) acc[i][x] = fmaf(wk, v[i][k][x], acc[i][x]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (i < rows) attn_merge_store<D>(a, it, r0 + i, V * lane, acc[i], dark[i] && L[i] == 0.f ? __int_as_float(0x7fffffff) : L[i]);
}

// Few rows: block (c, y) takes rows y, y + 8, ... of the item. A handful of parts: a warp to a row. Hundreds (a long sequence): the eight
// warps share a row, each a run of its parts, the runs added in order (131,071 positions of two kv heads, 222 parts to a row: the join
// alone 150 us with one warp and one part at a time; 46.8 in all with four blocks to an item, 45 with eight; 64 sequences 87.6 and 89.3).
#define ATTN_MERGE_BLOCKS 8
template <int ROWS, int D>
__global__ void __launch_bounds__(256) attn_merge_few_kernel(const __grid_constant__ AttnArgs a, int ctas) {
    constexpr int V = D / 32, B = 8;
    __shared__ float sums[8][D + 1];                              // a warp's weighted sums, and its sum of weights
    __shared__ float tops[8];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int c = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const AttnItem it = attn_item(a.meta, c, ctas);
    const int rows = it.ntok * a.g;
    if (!it.n || (int)blockIdx.y >= rows) return;
    const size_t slot = attn_slot_floats(ROWS, D);
    const bool together = it.n > 16;
    const int lo = together ? it.n * warp / 8 : 0, hi = together ? it.n * (warp + 1) / 8 : it.n;
    auto part_of = [&](int k) { return a.part + ((size_t)(c + k) * 2 + (k == 0)) * slot; };
    // of the lane's parts lo + lane and lo + 32 + lane; a run has no more than 64 (ATTN_FEW_MAX)
    bool has[2];
    has[0] = lo + lane < hi && (together ? lo + lane == 0 || (a.meta[c + lo + lane].flags & ATTN_CONT) : it.flags != 0);
    has[1] = lo + 32 + lane < hi && (a.meta[c + lo + 32 + lane].flags & ATTN_CONT);
    for (int r = blockIdx.y + (together ? 0 : ATTN_MERGE_BLOCKS * warp); r < rows; r += ATTN_MERGE_BLOCKS * (together ? 1 : 8)) {
        float m[2], l[2], v[B][V];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float *p = part_of(lo + 32 * h + lane) + ROWS * D + r;
            m[h] = has[h] ? __ldcg(p) : -INFINITY;
            l[h] = has[h] ? __ldcg(p + ROWS) : 0.f;
        }
        auto rows_of = [&](int k0) {
#pragma unroll
            for (int k = 0; k < B; ++k)
                if (k0 + k < hi) attn_merge_load<D>(part_of(k0 + k) + (size_t)r * D + V * lane, v[k]);
        };
        rows_of(lo);
        float M = fmaxf(m[0], m[1]);
#pragma unroll
        for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
        if (together) {
            if (lane == 0) tops[warp] = M;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 8; ++i) M = fmaxf(M, tops[i]);
        }
        const bool dark = lo == 0 && __shfl_sync(0xffffffffu, l[0], 0) < 0.f;        // of the first part: every row that sees anything sees it
        const float mu = M == -INFINITY ? 0.f : M;
        const float w0 = exp2f(m[0] - mu), w1 = exp2f(m[1] - mu);
        float L = 0.f, acc[V] = {};
        for (int k0 = 0; lo + k0 < hi; k0 += B) {
            if (k0) rows_of(lo + k0);
#pragma unroll
            for (int k = 0; k < B; ++k) {
                const float wk = __shfl_sync(0xffffffffu, k0 < 32 ? w0 : w1, (k0 + k) & 31);
                const float lk = __shfl_sync(0xffffffffu, k0 < 32 ? l[0] : l[1], (k0 + k) & 31);
                if (lo + k0 + k >= hi || lk <= 0.f) continue;     // the part holds nothing of the row, perhaps not even numbers
                L = fmaf(wk, lk, L);
#pragma unroll
                for (int x = 0; x < V; ++x) acc[x] = fmaf(wk, v[k][x], acc[x]);
            }
        }
        if (together) {
#pragma unroll
            for (int x = 0; x < V; ++x) sums[warp][V * lane + x] = acc[x];
            if (lane == 0) sums[warp][D] = L;
            __syncthreads();
            if (warp == 0) {
#pragma unroll
                for (int i = 1; i < 8; ++i) {
#pragma unroll
                    for (int x = 0; x < V; ++x) acc[x] += sums[i][V * lane + x];
                    L += sums[i][D];
                }
            }
        }
        if (!together || warp == 0) attn_merge_store<D>(a, it, r, V * lane, acc, dark && L == 0.f ? __int_as_float(0x7fffffff) : L);
        if (together) __syncthreads();                            // sums and tops are read
    }
}

int attn_launch_merge(jl_ctx *ctx, const AttnArgs &a, int rows, int ctas, int unit, cudaStream_t s) {
    // Sequences that can be no longer than a unit leave no parts: 10.7 us instead of 16 for a prompt of seven tokens.
    if ((a.table ? (long long)a.max_pages << a.page_shift : (long long)a.total) <= unit) return JL_OK;
    const dim3 few(ctas, ATTN_MERGE_BLOCKS), many(ctas, rows / (8 * ATTN_MERGE_ROWS));
    const cudaError_t e = rows == ATTN_FEW_ROWS
        ? (a.d == 128 ? attn_launch_pdl(ctx, attn_merge_few_kernel<ATTN_FEW_ROWS, 128>, few, dim3(256), 0, s, a, ctas)
                      : attn_launch_pdl(ctx, attn_merge_few_kernel<ATTN_FEW_ROWS, 64>, few, dim3(256), 0, s, a, ctas))
        : (a.d == 128 ? attn_launch_pdl(ctx, attn_merge_many_kernel<128>, many, dim3(256), 0, s, a, ctas, rows)
                      : attn_launch_pdl(ctx, attn_merge_many_kernel<64>, many, dim3(256), 0, s, a, ctas, rows));
    JL_CUDA(ctx, e);
    ctx->st.launches++;
    return JL_OK;
}

// ------------------------------------------------------------------ the cache's writer
// Row r of qkv is a new token of the sequence it lies in; four consecutive values of it (two pairs) to a thread. Bound by bytes:
// qkv is read once, q_out and the pages written once. 4096 rows of 48 heads of 128 f32, 154 MB: 28 us, 5.5 TB/s; 64 rows: 4.4 us, latency.
__device__ __forceinline__ float4 attn_load4(const void *x, int dtype, size_t at) {
    if (dtype == JL_DT_F32) return __ldcs(reinterpret_cast<const float4 *>(static_cast<const float *>(x) + at));
    const uint2 w = __ldcs(reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(x) + at));
    if (dtype == JL_DT_BF16)
        return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xFFFF0000u), __uint_as_float(w.y << 16),
                           __uint_as_float(w.y & 0xFFFF0000u));
    const float2 p = __half22float2(*reinterpret_cast<const __half2 *>(&w.x)), q = __half22float2(*reinterpret_cast<const __half2 *>(&w.y));
    return make_float4(p.x, p.y, q.x, q.y);
}

struct AppendArgs {
    void *q_out, *k, *v;
    const void *qkv;
    const int *starts, *lens, *table;
    const float *cos_t, *sin_t;
    long long kv_tok, kv_head, kv_page;
    int nseq, total, hq, hkv, d, page_shift, n_pages, max_pages, max_pos, x_dtype, dtype;
};

__global__ void __launch_bounds__(256) attn_append_kernel(const __grid_constant__ AppendArgs a) {
    __shared__ int sh[2];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int row = blockIdx.x;
    if (threadIdx.x == 0) {
        int lo = 0, hi = a.nseq;                       // the last sequence that starts at or before the row: among equal starts the
        while (lo < hi) {                              // one that has rows
            const int mid = (lo + hi) >> 1;
            if (a.starts[mid + 1] <= row) lo = mid + 1; else hi = mid;
        }
        int page = -1, pos = -1;
        if (lo < a.nseq && row >= a.starts[lo]) {
            const long long p = (long long)a.lens[lo] - a.starts[lo + 1] + row;
            if (p >= 0 && p < a.max_pos && p < ((long long)a.max_pages << a.page_shift)) {
                pos = (int)p;
                page = a.table[(long long)lo * a.max_pages + (pos >> a.page_shift)];
                if ((unsigned)page >= (unsigned)a.n_pages) page = -1;
            }
        }
        sh[0] = pos; sh[1] = page;
    }
    __syncthreads();
    const int pos = sh[0], page = sh[1];
    if (pos < 0) return;
    const int heads = a.hq + 2 * a.hkv, quads = a.d / 4;
    const long long at = page * a.kv_page + (pos & ((1 << a.page_shift) - 1)) * a.kv_tok;
    for (int i = threadIdx.x; i < heads * quads; i += 256) {
        const int hd = i / quads, j = i - hd * quads;
        float4 v = attn_load4(a.qkv, a.x_dtype, ((size_t)row * heads + hd) * a.d + 4 * j);
        if (hd < a.hq + a.hkv) {
            const float2 c = reinterpret_cast<const float2 *>(a.cos_t + (size_t)pos * (a.d / 2))[j];
            const float2 s = reinterpret_cast<const float2 *>(a.sin_t + (size_t)pos * (a.d / 2))[j];
            v = make_float4(v.x * c.x - v.y * s.x, v.x * s.x + v.y * c.x, v.z * c.y - v.w * s.y, v.z * s.y + v.w * c.y);
        }
        if (hd < a.hq) {
            attn_store4(a.q_out, a.dtype, ((size_t)row * a.hq + hd) * a.d + 4 * j, v);
        } else if (page >= 0) {
            const bool isk = hd < a.hq + a.hkv;
            attn_store4(isk ? a.k : a.v, a.dtype, (size_t)(at + (long long)(hd - a.hq - (isk ? 0 : a.hkv)) * a.kv_head + 4 * j), v);
        }
    }
}

// ------------------------------------------------------------------ C ABI
namespace {
// The caller's current device comes back however the call ends.
struct DeviceGuard {
    int was, to;
    bool ok;
    explicit DeviceGuard(int device) : was(-1), to(device), ok(false) {
        if (cudaGetDevice(&was) != cudaSuccess) { cudaGetLastError(); was = -1; }
        ok = was == device || cudaSetDevice(device) == cudaSuccess;
        if (!ok) cudaGetLastError();
    }
    ~DeviceGuard() { if (was >= 0 && was != to) cudaSetDevice(was); }
};
bool off16(const void *p) { return ((uintptr_t)p & 15u) != 0; }
bool is16(int dtype) { return dtype == JL_DT_F16 || dtype == JL_DT_BF16; }

// What both attention calls ask of their arguments; JL_OK, or the status with its reason.
int check_common(jl_ctx *ctx, const char *name, const void *out, int out_dtype, const void *q, const void *k, const void *v, int dtype,
                 long long q_tok, long long q_head, const void *starts, int nseq, int total, int hq, int hkv, int d, float scale,
                 const void *scratch, size_t scratch_bytes) {
    if (!out || !q || !k || !v || !starts || !scratch) return jl_set_err(ctx, JL_EINVAL, "%s: a pointer is NULL", name);
    if (!is16(dtype)) return jl_set_err(ctx, JL_EINVAL, "%s: q, k and v are f16 or bf16", name);
    if (out_dtype != JL_DT_F32 && !is16(out_dtype)) return jl_set_err(ctx, JL_EINVAL, "%s: out is f32, f16 or bf16", name);
    if (nseq < 1 || total < 1 || hq < 1 || hkv < 1) return jl_set_err(ctx, JL_EINVAL, "%s: sizes below one", name);
    if (hq % hkv || hq / hkv > 16) return jl_set_err(ctx, JL_ENOTSUP, "%s: %d query heads over %d kv heads (a multiple, up to 16)", name, hq, hkv);
    if (d != 64 && d != 128) return jl_set_err(ctx, JL_ENOTSUP, "%s: head size %d (64 and 128 are served)", name, d);
    if (!(scale > 0.f) || !(scale * 1.4426950408889634f < INFINITY)) return jl_set_err(ctx, JL_EINVAL, "%s: the scale must be positive and finite", name);
    if (total > (1 << 26) || hq > 1024 || nseq > (1 << 20)) return jl_set_err(ctx, JL_ENOTSUP, "%s: too many rows, heads or sequences", name);
    if (off16(out) || off16(q) || off16(k) || off16(v) || off16(scratch) || ((uintptr_t)starts & 3))
        return jl_set_err(ctx, JL_EINVAL, "%s: pointers must be 16-byte aligned (4 for the sequences' tables)", name);
    if (q_tok < 0 || q_head < 0 || q_tok % 8 || q_head % 8 || q_tok >= (1ll << 31) || q_head >= (1ll << 31))
        return jl_set_err(ctx, JL_EINVAL, "%s: strides of q must be multiples of 8 elements", name);
    if (scratch_bytes < jl_attn_scratch_bytes(ctx)) return jl_set_err(ctx, JL_EINVAL, "%s: scratch of %zu bytes, jl_attn_scratch_bytes is %zu", name, scratch_bytes, jl_attn_scratch_bytes(ctx));
    return JL_OK;
}

// Sequences of up to max_new new rows: those of at most sixteen query rows to a kv head go to the kernel that takes sixteen, the others
// to the tensor core's 256. A launch that finds no sequence of its own costs about 4 us: there are two only where `mixed` says that both
// kinds are likely.
int attn_launch(jl_ctx *ctx, AttnArgs a, int dtype, long long max_new, bool mixed, cudaStream_t s) {
    a.row_lo = 0;
    a.row_hi = INT_MAX;
    if (max_new * a.g <= ATTN_FEW_ROWS) return attn_launch_few(ctx, a, dtype, s);
    if (mixed) {
        a.row_hi = ATTN_FEW_ROWS;
        const int rc = attn_launch_few(ctx, a, dtype, s);
        if (rc != JL_OK) return rc;
        a.row_lo = a.row_hi;
        a.row_hi = INT_MAX;
    }
    return attn_launch_tc5(ctx, a, dtype, max_new * a.g, s);
}

// A cache in pages: JL_OK, or the status with its reason. *shift: log2 of the page length.
int check_pages(jl_ctx *ctx, const char *name, const jl_paged_kv *kv, jl_paged_kv *out, int *shift) {
    if (!kv || kv->struct_size < sizeof(jl_paged_kv)) return jl_set_err(ctx, JL_EINVAL, "%s: a jl_paged_kv with its struct_size set", name);
    *out = *kv;
    if (!kv->k || !kv->v || !kv->page_table) return jl_set_err(ctx, JL_EINVAL, "%s: a pointer of the cache is NULL", name);
    if (!is16(kv->dtype)) return jl_set_err(ctx, JL_EINVAL, "%s: the cache is f16 or bf16", name);
    if (kv->n_kv < 1 || kv->n_pages < 1 || kv->n_seq < 1 || kv->max_pages < 1) return jl_set_err(ctx, JL_EINVAL, "%s: sizes below one", name);
    int s = 0;
    while (s < 11 && (1 << s) < kv->page_len) s++;
    if (kv->page_len < 16 || kv->page_len > 1024 || (1 << s) != kv->page_len)
        return jl_set_err(ctx, JL_ENOTSUP, "%s: pages of %d positions (powers of two from 16 to 1024 are served)", name, kv->page_len);
    if (((long long)kv->max_pages << s) > (1ll << 30)) return jl_set_err(ctx, JL_ENOTSUP, "%s: more than 2^30 positions to a sequence", name);
    if (off16(kv->k) || off16(kv->v) || ((uintptr_t)kv->page_table & 3)) return jl_set_err(ctx, JL_EINVAL, "%s: the pages must be 16-byte aligned", name);
    *shift = s;
    return JL_OK;
}
}  // namespace

JL_EXPORT size_t jl_attn_scratch_bytes(jl_ctx *ctx) {
    if (!ctx) return 0;
    const int few = attn_few_grid(ctx);
    const size_t f = (size_t)few * 2 * attn_slot_floats(ATTN_FEW_ROWS, 128), t = (size_t)ctx->sm_count * 2 * attn_slot_floats(ATTN_TC_ROWS, 128);
    return attn_meta_bytes(few) + (f > t ? f : t) * sizeof(float);
}

JL_EXPORT int jl_attn_prompt(jl_ctx *ctx, void *out, int out_dtype, const void *q, long long q_tok_stride, long long q_head_stride,
                             const void *k, const void *v, long long kv_tok_stride, long long kv_head_stride, int dtype,
                             const int32_t *starts_dev, int nseq, int total, int hq, int hkv, int d, float scale, void *scratch,
                             size_t scratch_bytes, void *stream) {
    if (!ctx) return JL_EINVAL;
    std::lock_guard<std::mutex> lk(ctx->mu);
    int rc = check_common(ctx, "jl_attn_prompt", out, out_dtype, q, k, v, dtype, q_tok_stride, q_head_stride, starts_dev, nseq, total, hq,
                          hkv, d, scale, scratch, scratch_bytes);
    if (rc != JL_OK) return rc;
    if (kv_tok_stride < 0 || kv_head_stride < 0 || kv_tok_stride % 8 || kv_head_stride % 8 || kv_tok_stride >= (1ll << 31) ||
        kv_head_stride >= (1ll << 38))
        return jl_set_err(ctx, JL_EINVAL, "jl_attn_prompt: strides of k and v must be multiples of 8 elements");
    if (ctx->unhealthy) return jl_set_err(ctx, JL_ECUDA, "context is unhealthy after an earlier CUDA error");
    DeviceGuard dg(ctx->device);
    if (!dg.ok) return jl_set_err(ctx, JL_ECUDA, "jl_attn_prompt: the device cannot be made current");
    AttnArgs a = {};
    a.out = out; a.q = q; a.k = k; a.v = v; a.starts = starts_dev;
    a.q_tok = q_tok_stride; a.q_head = q_head_stride; a.kv_tok = kv_tok_stride; a.kv_head = kv_head_stride;
    a.nseq = nseq; a.total = total; a.hq = hq; a.hkv = hkv; a.g = hq / hkv; a.d = d;
    a.out_dtype = out_dtype; a.scale_log2 = scale * 1.4426950408889634f; a.status = ctx->dev_status;
    a.meta = static_cast<AttnMeta *>(scratch);
    a.part = reinterpret_cast<float *>(static_cast<uint8_t *>(scratch) + attn_meta_bytes(attn_few_grid(ctx)));
    rc = attn_launch(ctx, a, dtype, total, false, (cudaStream_t)stream);
    if (rc == JL_OK) ctx->st.served++;
    return rc;
}

JL_EXPORT int jl_attn_paged(jl_ctx *ctx, void *out, int out_dtype, const void *q, long long q_tok_stride, long long q_head_stride,
                            const jl_paged_kv *kv, const int32_t *starts_dev, const int32_t *lens_dev, int total, int max_new, int hq,
                            float scale, void *scratch, size_t scratch_bytes, void *stream) {
    if (!ctx) return JL_EINVAL;
    std::lock_guard<std::mutex> lk(ctx->mu);
    jl_paged_kv c;
    int shift = 0, rc = check_pages(ctx, "jl_attn_paged", kv, &c, &shift);
    if (rc == JL_OK)
        rc = check_common(ctx, "jl_attn_paged", out, out_dtype, q, c.k, c.v, c.dtype, q_tok_stride, q_head_stride, starts_dev, c.n_seq, total,
                          hq, c.n_kv, c.head_dim, scale, scratch, scratch_bytes);
    if (rc != JL_OK) return rc;
    if (!lens_dev || ((uintptr_t)lens_dev & 3)) return jl_set_err(ctx, JL_EINVAL, "jl_attn_paged: the sequences' lengths are missing or misaligned");
    if (max_new < 1) return jl_set_err(ctx, JL_EINVAL, "jl_attn_paged: max_new below one");
    if (ctx->unhealthy) return jl_set_err(ctx, JL_ECUDA, "context is unhealthy after an earlier CUDA error");
    DeviceGuard dg(ctx->device);
    if (!dg.ok) return jl_set_err(ctx, JL_ECUDA, "jl_attn_paged: the device cannot be made current");
    AttnArgs a = {};
    a.out = out; a.q = q; a.k = c.k; a.v = c.v; a.starts = starts_dev; a.lens = lens_dev; a.table = c.page_table;
    a.q_tok = q_tok_stride; a.q_head = q_head_stride;
    a.kv_tok = c.head_dim; a.kv_head = (long long)c.page_len * c.head_dim; a.kv_page = a.kv_head * c.n_kv;
    a.nseq = c.n_seq; a.total = total; a.hq = hq; a.hkv = c.n_kv; a.g = hq / c.n_kv; a.d = c.head_dim;
    a.page_shift = shift; a.n_pages = c.n_pages; a.max_pages = c.max_pages;
    a.out_dtype = out_dtype; a.scale_log2 = scale * 1.4426950408889634f; a.status = ctx->dev_status;
    a.meta = static_cast<AttnMeta *>(scratch);
    a.part = reinterpret_cast<float *>(static_cast<uint8_t *>(scratch) + attn_meta_bytes(attn_few_grid(ctx)));
    rc = attn_launch(ctx, a, c.dtype, max_new, c.n_seq > 1 && total < (long long)max_new * c.n_seq, (cudaStream_t)stream);
    if (rc == JL_OK) ctx->st.served++;
    return rc;
}

JL_EXPORT int jl_rope_append(jl_ctx *ctx, void *q_out, const void *qkv, int x_dtype, const jl_paged_kv *kv, const int32_t *starts_dev,
                             const int32_t *lens_dev, int total, int hq, const float *cos_t, const float *sin_t, int max_pos, void *stream) {
    if (!ctx) return JL_EINVAL;
    std::lock_guard<std::mutex> lk(ctx->mu);
    jl_paged_kv c;
    int shift = 0, rc = check_pages(ctx, "jl_rope_append", kv, &c, &shift);
    if (rc != JL_OK) return rc;
    if (!q_out || !qkv || !starts_dev || !lens_dev || !cos_t || !sin_t) return jl_set_err(ctx, JL_EINVAL, "jl_rope_append: a pointer is NULL");
    if (x_dtype != JL_DT_F32 && !is16(x_dtype)) return jl_set_err(ctx, JL_EINVAL, "jl_rope_append: qkv is f32, f16 or bf16");
    if (total < 1 || hq < 1 || max_pos < 1) return jl_set_err(ctx, JL_EINVAL, "jl_rope_append: sizes below one");
    if (c.head_dim < 4 || c.head_dim > 1024 || c.head_dim % 4) return jl_set_err(ctx, JL_ENOTSUP, "jl_rope_append: head size %d (a multiple of 4)", c.head_dim);
    if (total > (1 << 26) || hq > 1024 || c.n_kv > 1024) return jl_set_err(ctx, JL_ENOTSUP, "jl_rope_append: too many rows or heads");
    if (off16(q_out) || off16(qkv) || off16(cos_t) || off16(sin_t) || ((uintptr_t)starts_dev & 3) || ((uintptr_t)lens_dev & 3))
        return jl_set_err(ctx, JL_EINVAL, "jl_rope_append: pointers must be 16-byte aligned (4 for the sequences' tables)");
    if (ctx->unhealthy) return jl_set_err(ctx, JL_ECUDA, "context is unhealthy after an earlier CUDA error");
    DeviceGuard dg(ctx->device);
    if (!dg.ok) return jl_set_err(ctx, JL_ECUDA, "jl_rope_append: the device cannot be made current");
    AppendArgs a = {};
    a.q_out = q_out; a.k = c.k; a.v = c.v; a.qkv = qkv; a.starts = starts_dev; a.lens = lens_dev; a.table = c.page_table;
    a.cos_t = cos_t; a.sin_t = sin_t;
    a.kv_tok = c.head_dim; a.kv_head = (long long)c.page_len * c.head_dim; a.kv_page = a.kv_head * c.n_kv;
    a.nseq = c.n_seq; a.total = total; a.hq = hq; a.hkv = c.n_kv; a.d = c.head_dim; a.page_shift = shift; a.n_pages = c.n_pages;
    a.max_pages = c.max_pages; a.max_pos = max_pos; a.x_dtype = x_dtype; a.dtype = c.dtype;
    const cudaError_t e = attn_launch_pdl(ctx, attn_append_kernel, dim3(total), dim3(256), 0, (cudaStream_t)stream, a);
    JL_CUDA(ctx, e);
    ctx->st.launches++;
    ctx->st.served++;
    return JL_OK;
}

// How a launch divides the work, on the host: the segments of CTA `cta` as (sequence, block, head, first unit, end unit, units of the
// item). The items, the cuts and the walk are the device's own functions (attn.cuh); only the search for the sequences that the cuts
// fall into is the host's, one sequence after the other where a warp looks at 32 (attn_share). Test-only.
JL_EXPORT int jl_test_attn_share_as(const int32_t *starts, const int32_t *lens, int nseq, int total, int hkv, int g, int row_lo, int row_hi,
                                    int tok_item, int item_cost, int snap, int unit_shift, int min_units, int page_shift, int max_pages,
                                    int grid, int cta, int32_t *segs, int cap) {
    if (!starts || !segs || nseq < 1 || hkv < 1 || g < 1 || tok_item < 1 || item_cost < 0 || snap < 0 || unit_shift < 1 || unit_shift > 16 ||
        min_units < 1 || page_shift < 0 || page_shift > 16 || grid < 1 || cta < 0 || cta >= grid)
        return JL_EINVAL;
    AttnArgs a = {};
    a.starts = starts; a.lens = lens; a.nseq = nseq; a.total = total; a.hkv = hkv; a.tok_item = tok_item;
    a.table = max_pages > 0 ? starts : nullptr;       // only its presence matters here
    a.page_shift = page_shift; a.max_pages = max_pages;
    a.g = g; a.row_lo = row_lo; a.row_hi = row_hi; a.item_cost = item_cost; a.snap = snap;
    AttnCut first, last;
    attn_share_host(a, cta, grid, unit_shift, min_units, first, last);
    AttnWalk w;
    w.begin(first, last);
    AttnSeg sg;
    int n = 0;
    while (w.next(a, unit_shift, sg)) {
        if (n == cap) return -100;
        int32_t *o = segs + 6 * n++;
        o[0] = sg.seq; o[1] = sg.blk; o[2] = sg.head; o[3] = sg.u0; o[4] = sg.u1; o[5] = sg.units;
    }
    return n;
}
JL_EXPORT int jl_test_attn_share(const int32_t *starts, const int32_t *lens, int nseq, int total, int hkv, int tok_item, int unit_shift,
                                 int min_units, int page_shift, int max_pages, int grid, int cta, int32_t *segs, int cap) {
    return jl_test_attn_share_as(starts, lens, nseq, total, hkv, 1, 0, INT_MAX, tok_item, 1, 2, unit_shift, min_units, page_shift, max_pages,
                                 grid, cta, segs, cap);
}
