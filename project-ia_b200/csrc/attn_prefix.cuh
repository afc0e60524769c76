// attn_prefix.cuh — attention of a batch's new tokens over a shared prefix
// and each sequence's own paged rows (q_b200_attn_prefix).
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(y_j - m),  y_j = scale log2(e) q.k_j
//
// over the rows j that the token sees, in one pass: a running reference m near
// the maximum and sum l, and the accumulated output multiplied by 2^(m_old -
// m_new) when m moves.  The rows may be cut into parts that different CTAs take; a part
// leaves (m, l, o) in fp32 in the workspace and attn_join_kernel adds them
// in part order (the same result on every run).
//
// This file holds what the passes share, and attn_rows_kernel, the pass for
// more than 32 vectors of a KV head where tcgen05 is not used (fp32 caches,
// head_dim 32, a scale that is not positive, a prompt's own rows).  One CTA
// takes 64 query vectors (tokens x the G heads that share a KV head), 16 for
// each of four warps, and a range of rows in tiles that a fifth warp brings
// into a ring with cp.async; a row's page is looked up by one lane, so pages
// may have any size and end anywhere in a tile.  Products are mma.sync:
// m16n8k16 for fp16 and bf16; for fp32 m16n8k8 tf32 on halves v = hi + lo of
// 11 bits each, hi.hi + hi.lo + lo.hi (the dropped lo.lo is 2^-22 relative),
// with the hi.hi sums folded into fp32 every few products because the tensor
// core truncates when it accumulates (errors against 64 bits come out at
// 4e-7, half of an fp32 product's).  P is rounded to the cache's type for P.V
// (fp16, bf16), as the products' operand type asks: an error of the size of the
// result's own rounding (with it 1.3 to 1.45 times the error against 64 bits
// of a result that is rounded once).  l sums what is multiplied here and in
// attn_few_kernel, the weights before their rounding in the tcgen05 pass.
//
// Bound: the products (64 vectors a row of K and V).
#pragma once

#include <type_traits>

#include "rotate.cuh"

namespace qb200 {

struct PrefixArgs {
    const void* q;
    void* out;
    const void* k;
    const void* v;
    uint64_t q_token, q_head, o_token, o_head;
    uint64_t page_stride, head_stride, row_stride;
    const uint32_t* q_start;
    const uint32_t* pages;
    const uint32_t* lens;
    const uint32_t* prefix_pages;
    const uint32_t* prefix_len;
    float* part_o;    // [parts][n_tokens][n_heads][HD]
    float2* part_ml;  // [parts][n_tokens][n_heads]
    FastDiv page_rows, by_group;
    uint32_t n_pages, pages_per_seq, n_tokens, n_seqs, n_heads, group;
    uint32_t max_q, max_len, max_prefix;
    uint32_t tiles;      // row tiles of an item (prefix: of all tokens; own: of one sequence)
    uint32_t splits;     // parts that an item's rows are cut into
    uint32_t part0;      // this launch's first part
    uint32_t last;       // 1: writes out itself, after `merge` parts of the pass before it
    uint32_t merge;
    uint32_t n_parts;    // of the join
    uint32_t first;      // waits for the stream's work before it; a later pass reads the call's inputs at once
    uint32_t cluster;    // attn_few_kernel: the splits are a cluster's
    uint32_t alternate;  // tcgen05 pass: one tile of vectors, even and odd row tiles
    uint32_t shared;     // 1: the prefix for all tokens; 0: per sequence
    uint32_t with_prefix;  // own pass: the prefix's rows come before the own ones
    float c;             // scale * log2(e)
};

template <typename T>
struct AttnTraits;
template <>
struct AttnTraits<__half> {
    static constexpr int KT = 64, STAGES = 3;
};
template <>
struct AttnTraits<__nv_bfloat16> {
    static constexpr int KT = 64, STAGES = 3;
};
template <>
struct AttnTraits<float> {
    static constexpr int KT = 32, STAGES = 3;
};

static constexpr uint32_t ATTN_CONSUMERS = 128;  // four warps that multiply, one that copies
static constexpr uint32_t ATTN_THREADS = 160;
static constexpr uint32_t ATTN_MAX_PARTS = 128;
static constexpr uint32_t ATTN_VECS = 64;  // of a CTA of attn_rows_kernel

template <typename T, int HD>
constexpr size_t attn_rows_smem() {
    constexpr size_t ring = (size_t)AttnTraits<T>::STAGES * AttnTraits<T>::KT * HD * sizeof(T) * 2 + ATTN_VECS * HD * sizeof(T);
    constexpr size_t out = ATTN_VECS * (HD + 4 + 2) * 4;
    return ring > out ? ring : out;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Arrives on `bar` once every copy that this thread has issued so far is done.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Weights are 2^(y - m) for a reference m that moves only when the largest
// score y exceeds it by LIFT + 8, and then to LIFT below that score: few
// outputs are rescaled, and the quotient o / l is the same.  fp16 loses bits
// of weights below 2^-14 and all of 2^-25 (thousands of rows far below one
// that outweighs each of them can still be the result), so they lie as high as
// its range has room for the largest, at 2^7 to 2^15; bf16 and fp32 have the
// exponents, and weights of at most 1 keep sums of great values finite.
template <typename T>
constexpr float ATTN_LIFT = std::is_same<T, __half>::value ? 7.0f : -8.0f;
template <typename T>
__device__ __forceinline__ float attn_reference(float m, float top) {
    return top > m + (ATTN_LIFT<T> + 8.0f) ? top - ATTN_LIFT<T> : m;
}

// Barrier of the consumer warps alone.
__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ bool consumers_or(bool v) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred.aligned q, 1, 128, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"((uint32_t)v)
        : "memory");
    return r != 0;
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}

__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// v = hi + lo: hi of 11 significant bits rounded to nearest, lo the rest, of
// which the tensor core reads the upper 19 bits (all but the last bit of the
// 12 it can have).  hi stays finite: v near the type's largest would be
// rounded to infinity, whose product with a weight of zero is no number.  So
// an infinity or a NaN (whose bits the rounding could carry into the sign) is
// in lo alone, and reaches the sum from there.
__device__ __forceinline__ void split_tf32(uint32_t v, uint32_t& hi, uint32_t& lo) {
    float c;
    asm("min.xorsign.abs.f32 %0, %1, %2;" : "=f"(c) : "f"(__uint_as_float(v)), "f"(__uint_as_float(0x7f7fe000u)));
    hi = (__float_as_uint(c) + 0x1000u) & 0xffffe000u;
    lo = __float_as_uint(__uint_as_float(v) - __uint_as_float(hi));
}

// 16-byte chunk c of row r in a tile of HD-wide rows: chunks are exchanged
// within 128 bytes so that 8 rows' equal chunks lie in 8 different banks
// groups.  Rows of 64 bytes (two to a bank line) turn every second row.
template <typename T, int HD>
__device__ __forceinline__ uint32_t tile_off(uint32_t r, uint32_t c) {
    constexpr uint32_t RB = HD * sizeof(T);
    if constexpr (RB >= 128) return r * RB + ((c ^ (r & 7)) << 4);
    else return r * RB + ((c ^ ((r >> 1) & 3)) << 4);
}
// fp32 values are read element by element along rows 2t, 2t+1: rows 0, 2, 4,
// 6 have to differ by two chunks.
template <int HD>
__device__ __forceinline__ uint32_t v32_off(uint32_t r, uint32_t c) {
    return r * HD * 4 + ((c ^ (((r >> 1) & 3) << 1)) << 4);
}

template <typename T, int HD>
__device__ __forceinline__ uint32_t vt_off(uint32_t r, uint32_t c) {
    if constexpr (sizeof(T) == 4) return v32_off<HD>(r, c);
    else return tile_off<T, HD>(r, c);
}
// Whether the 16 bytes at a shared address hold finite numbers only.
template <typename T>
__device__ __forceinline__ bool finite16(uint32_t addr) {
    uint32_t x[4];
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(addr));
    constexpr uint32_t E = sizeof(T) == 4 ? 0x7f800000u : 0u;
    bool ok = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (E != 0u) {
            ok &= (x[i] & E) != E;
        } else {
            constexpr uint32_t lo = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
            ok &= (x[i] & lo) != lo && (x[i] & (lo << 16)) != (lo << 16);
        }
    }
    return ok;
}

// What a CTA has to do.
struct AttnItem {
    uint32_t tok0, n_tok;   // tokens that its vectors come from
    uint32_t vec0, n_vec;   // vectors (token, head in group) of this tile
    uint32_t seq;           // own rows of this sequence
    uint32_t n_prefix;      // rows 0..n_prefix-1 are the prefix's
    uint32_t n_rows;        // all rows
    uint32_t r0, r1;        // this part's
    int32_t see0;           // vector of token i sees rows < see0 + i (own), all when >= n_rows
};

__device__ __forceinline__ bool attn_item(const PrefixArgs& a, uint32_t item, uint32_t split, uint32_t vecs, uint32_t step,
                                          AttnItem& w) {
    // all loads first: they are the start of every CTA's chain
    uint32_t tile = item, P = 0, L = 0, s0 = 0, s1 = 0;
    w.seq = 0;
    if ((a.shared || a.with_prefix) && a.prefix_pages) P = __ldg(a.prefix_len);
    if (!a.shared) {
        w.seq = item / a.tiles;
        tile = item - w.seq * a.tiles;
        L = __ldg(a.lens + w.seq);
        if (a.q_start) {
            s0 = __ldg(a.q_start + w.seq);
            s1 = __ldg(a.q_start + w.seq + 1);
        } else {
            s0 = w.seq;
            s1 = s0 + 1;
        }
    }
    const bool bad = s0 > s1 || s1 > a.n_tokens || s1 - s0 > a.max_q;
    if (P > a.max_prefix || L > a.max_len || bad) {
        qdev_fail(QDEV_BAD_ARG);
        P = min(P, a.max_prefix);
        L = min(L, a.max_len);
    }
    w.tok0 = a.shared ? 0 : s0;
    w.n_tok = a.shared ? a.n_tokens : bad ? 0 : s1 - s0;
    w.see0 = a.shared ? 0x40000000 : (int32_t)(P + L) - (int32_t)w.n_tok + 1;
    w.n_prefix = P;
    w.n_rows = P + L;
    w.vec0 = tile * vecs;
    const uint32_t all = w.n_tok * a.group;
    if (w.vec0 >= all) return false;
    w.n_vec = min(vecs, all - w.vec0);
    const uint32_t chunk = ((w.n_rows + a.splits - 1) / a.splits + step - 1) / step * step;
    w.r0 = min(split * chunk, w.n_rows);
    w.r1 = min(w.r0 + chunk, w.n_rows);
    return true;
}

// The page that row r of the item lies in, as the table has it.
__device__ __forceinline__ uint32_t attn_page(const PrefixArgs& a, const AttnItem& w, uint32_t r) {
    const bool pre = r < w.n_prefix;
    const uint32_t pi = fast_div(pre ? r : r - w.n_prefix, a.page_rows);
    return __ldg(pre ? a.prefix_pages + pi : a.pages + (size_t)w.seq * a.pages_per_seq + pi);
}
// Offset of row r in its page (elements); ~0 where the page is not one.
__device__ __forceinline__ uint64_t attn_offset(const PrefixArgs& a, const AttnItem& w, uint32_t head, uint32_t r, uint32_t page) {
    if (page >= a.n_pages) {
        qdev_fail(QDEV_BAD_ARG);
        return ~0ull;
    }
    const uint32_t i = r < w.n_prefix ? r : r - w.n_prefix;
    return page * a.page_stride + head * a.head_stride + (uint64_t)(i - fast_div(i, a.page_rows) * a.page_rows.d) * a.row_stride;
}
__device__ __forceinline__ bool attn_row(const PrefixArgs& a, const AttnItem& w, uint32_t head, uint32_t r, uint64_t& off) {
    off = attn_offset(a, w, head, r, attn_page(a, w, r));
    return off != ~0ull;
}

// Sum of parts (m, l, o) for four outputs of a vector.
template <int HD>
struct PartSum {
    float M = -INFINITY, L = 0.0f;
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    // Weights 2^(m - M); a part without a row (m = -inf, l = 0, o = 0) or
    // with NaN sums is added as it is.
    template <int N>
    __device__ __forceinline__ void add(const float2 (&ml)[N], const float4 (&y)[N]) {
        float top = M;
#pragma unroll
        for (int k = 0; k < N; ++k) top = fmaxf(top, ml[k].x);
        const float f0 = M == top ? 1.0f : ex2(M - top);
        M = top;
        L *= f0;
        x = make_float4(x.x * f0, x.y * f0, x.z * f0, x.w * f0);
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const float f = ml[k].x == top ? 1.0f : ex2(ml[k].x - top);
            L = fmaf(ml[k].y, f, L);
            x.x = fmaf(y[k].x, f, x.x);
            x.y = fmaf(y[k].y, f, x.y);
            x.z = fmaf(y[k].z, f, x.z);
            x.w = fmaf(y[k].w, f, x.w);
        }
    }
    // The workspace's first n parts of (token, head) id, twelve loads of each
    // kind under way at once.
    __device__ __forceinline__ void add_parts(const PrefixArgs& a, uint64_t id, uint32_t c, uint32_t n) {
        constexpr int N = 12;
        const uint64_t stride = (uint64_t)a.n_tokens * a.n_heads;
        const float4* po = reinterpret_cast<const float4*>(a.part_o) + id * (HD / 4) + c;
        for (uint32_t p = 0; p < n; p += N) {
            float2 ml[N];
            float4 y[N];
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const bool in = p + k < n;
                ml[k] = in ? __ldcg(a.part_ml + (p + k) * stride + id) : make_float2(-INFINITY, 0.0f);
                y[k] = in ? __ldcg(po + (p + k) * stride * (HD / 4)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
            add<N>(ml, y);
        }
    }
    template <typename T>
    __device__ __forceinline__ void store(const PrefixArgs& a, uint64_t tok, uint32_t h, uint32_t c) {
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
        float y[4] = {x.x * inv, x.y * inv, x.z * inv, x.w * inv};
        if (L == 0.0f) y[0] = y[1] = y[2] = y[3] = 0.0f;  // no row is seen
        store_vec<T, 4>(reinterpret_cast<T*>(a.out) + tok * a.o_token + (uint64_t)h * a.o_head + c * 4, y);
    }
};

template <typename T, int HD>
__global__ void __launch_bounds__(ATTN_THREADS) attn_rows_kernel(const __grid_constant__ PrefixArgs a) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int KT = AttnTraits<T>::KT, ST = AttnTraits<T>::STAGES;
    constexpr int NT = KT / 8, ND = HD / 8;        // score and output tiles of 8 columns
    constexpr int CH = HD * (int)sizeof(T) / 16;   // 16-byte chunks of a row
    constexpr int RP = 32 / CH;                    // rows that one copy instruction of the warp brings
    constexpr uint32_t TILE = KT * HD * sizeof(T);
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t full[ST], empty[ST];
    __shared__ bool s_bad[KT];
    const uint32_t s_kv = smem_u32(smem), s_q = s_kv + ST * 2 * TILE;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const uint32_t split = blockIdx.x, head = blockIdx.z;

    if (a.first) pdl_wait();
    pdl_trigger();  // the pass after this one may start beside it
    AttnItem w;
    if (!attn_item(a, blockIdx.y, split, ATTN_VECS, KT, w)) {
        pdl_wait();
        return;
    }
    if (tid == 0) {
        for (int i = 0; i < ST; ++i) {
            mbar_init(&full[i], 32);
            mbar_init(&empty[i], 4);
        }
        fence_mbar_init();
    }
    __syncthreads();
    const uint32_t n_tiles = (w.r1 - w.r0 + KT - 1) / KT;
    const T* kb = reinterpret_cast<const T*>(a.k);
    const T* vb = reinterpret_cast<const T*>(a.v);

    if (warp == 4) {
        // ---- producer: row offsets, one row (or two) of the tile per lane, then 16-byte copies ----
        const uint32_t lr = lane / CH, lc = lane % CH;
        for (uint32_t tile = 0; tile < n_tiles; ++tile) {
            const uint32_t slot = tile % ST, st = s_kv + slot * 2 * TILE;
            uint64_t off[KT / 32];
#pragma unroll
            for (int i = 0; i < KT / 32; ++i) {
                const uint32_t row = w.r0 + tile * KT + i * 32 + lane;
                if (!(row < w.r1 && attn_row(a, w, head, row, off[i]))) off[i] = ~0ull;  // zeros
            }
            if (tile >= ST && !__all_sync(0xffffffffu, mbar_wait(&empty[slot], (tile / ST - 1) & 1, QDEV_WAIT_EMPTY_TIMEOUT))) break;
#pragma unroll
            for (int p = 0; p < KT / RP; ++p) {
                const uint32_t r = p * RP + lr;
                const uint64_t o = __shfl_sync(0xffffffffu, off[p * RP / 32], r & 31);
                const uint32_t n = o == ~0ull ? 0u : 16u;
                const uint64_t at = (o == ~0ull ? 0ull : o) + lc * (16 / sizeof(T));
                cp_async16(st + tile_off<T, HD>(r, lc), kb + at, n);
                cp_async16(st + TILE + vt_off<T, HD>(r, lc), vb + at, n);
            }
            cp_async_arrive(&full[slot]);
        }
        cp_async_wait_all();
        pdl_wait();
        return;
    }

    // ---- consumers -------------------------------------------------------------------------------
    for (uint32_t e = tid; e < ATTN_VECS * CH; e += ATTN_CONSUMERS) {
        const uint32_t r = e / CH, c = e % CH;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < w.n_vec) {
            const uint32_t i = fast_div(w.vec0 + r, a.by_group), h = head * a.group + (w.vec0 + r - i * a.group);
            v = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.q) + (uint64_t)(w.tok0 + i) * a.q_token + h * a.q_head) + c);
        }
        *reinterpret_cast<uint4*>(smem + ST * 2 * TILE + tile_off<T, HD>(r, c)) = v;
    }
    consumers_sync();

    uint32_t qf[F32 ? 1 : HD / 16][4];
    if constexpr (!F32) {
#pragma unroll
        for (int j = 0; j < HD / 16; ++j)
            ldsm4(s_q + tile_off<T, HD>(warp * 16 + (lane & 15), 2 * j + (lane >> 4)), qf[j]);
    }

    // vectors g and g + 8 of this warp's 16: rows they see, running maximum and sum
    int32_t see[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t v = w.vec0 + warp * 16 + g + 8 * h;
        see[h] = w.see0 + (int32_t)fast_div(v, a.by_group);
        // tokens before the first own row see the prefix alone
        if (!a.shared) see[h] = max(see[h], (int32_t)w.n_prefix);
    }
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    float o[ND][4];
#pragma unroll
    for (int n = 0; n < ND; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;

    bool alive = true;
    for (uint32_t tile = 0; tile < n_tiles; ++tile) {
        // after a wait that ran out the others are not tried: every warp still meets every barrier
        if (alive) alive = __all_sync(0xffffffffu, mbar_wait(&full[tile % ST], (tile / ST) & 1, QDEV_WAIT_FULL_TIMEOUT));
        const uint32_t sk = s_kv + (tile % ST) * 2 * TILE, sv = sk + TILE;
        const uint32_t first = w.r0 + tile * KT;  // row of the tile's key 0

        // ---- scores -----------------------------------------------------------------
        float s[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
        if constexpr (!F32) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < HD / 32; ++j) {
                    uint32_t b[4];
                    ldsm4(sk + tile_off<T, HD>(n * 8 + (lane & 7), 4 * j + (lane >> 3)), b);
                    mma16(s[n], qf[2 * j], b[0], b[1], T());
                    mma16(s[n], qf[2 * j + 1], b[2], b[3], T());
                }
        } else {
            float sl[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) sl[n][0] = sl[n][1] = sl[n][2] = sl[n][3] = 0.0f;
#pragma unroll 2
            for (int j = 0; j < HD / 16; ++j) {  // two k8 steps
                uint32_t qh[2][4], ql[2][4];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    uint32_t q[4];
                    ldsm4(s_q + tile_off<T, HD>(warp * 16 + (lane & 15), 2 * (2 * j + e) + (lane >> 4)), q);
#pragma unroll
                    for (int i = 0; i < 4; ++i) split_tf32(q[i], qh[e][i], ql[e][i]);
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    uint32_t b[4], bh[4], bl[4];
                    ldsm4(sk + tile_off<T, HD>(n * 8 + (lane & 7), 4 * j + (lane >> 3)), b);
#pragma unroll
                    for (int i = 0; i < 4; ++i) split_tf32(b[i], bh[i], bl[i]);
                    float hh[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        mma8(hh, qh[e], bh[2 * e], bh[2 * e + 1]);
                        mma8(sl[n], qh[e], bl[2 * e], bl[2 * e + 1]);
                        mma8(sl[n], ql[e], bh[2 * e], bh[2 * e + 1]);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[n][i] += hh[i];
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[n][i] += sl[n][i];
        }

        // ---- mask, running maximum, exponentials ----------------------------------------
        const bool edge = first + KT > w.r1 || (int32_t)(first + KT) > w.see0;
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float y = s[n][i] * a.c;
                if (edge) {
                    const uint32_t row = first + n * 8 + 2 * t + (i & 1);
                    if (row >= w.r1 || (int32_t)row >= see[i >> 1]) y = -INFINITY;
                }
                s[n][i] = y;
                // a NaN score is carried into the sum, not into the maximum
                mx[i >> 1] = fmaxf(mx[i >> 1], y);
            }
        float corr[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
            const float M = attn_reference<T>(m[h], mx[h]);
            corr[h] = m[h] == M ? 1.0f : exp2f(m[h] - M);
            m[h] = M;
            l[h] *= corr[h];
        }
        uint32_t pf[F32 ? 1 : NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < 4; ++i) s[n][i] = s[n][i] == -INFINITY ? 0.0f : exp2f(s[n][i] - m[i >> 1]);
            if constexpr (!F32) {
                pf[n][0] = pack2<T>(s[n][0], s[n][1]);
                pf[n][1] = pack2<T>(s[n][2], s[n][3]);
                const float2 x = unpack2<T>(pf[n][0]), y = unpack2<T>(pf[n][1]);
                l[0] += x.x + x.y;
                l[1] += y.x + y.y;
            } else {
                l[0] += s[n][0] + s[n][1];
                l[1] += s[n][2] + s[n][3];
            }
        }

        // A row that only some of the tokens see may hold anything as far as the others are
        // concerned, and their weight 0 times an infinity or NaN in V would reach them: such
        // rows leave the tile and are added, where seen, after the product.
        const uint32_t hid0 = max((int32_t)first, w.see0), hid1 = min(first + KT, w.r1);
        bool bad = false;
        if (w.n_tok > 1 && !a.shared && hid0 < hid1) {
            for (uint32_t e = tid + (hid0 - first) * CH; e < (hid1 - first) * CH; e += ATTN_CONSUMERS)
                bad |= !finite16<T>(sv + vt_off<T, HD>(e / CH, e % CH));
            bad = consumers_or(bad);
            if (bad) {
                if (tid < KT) s_bad[tid] = false;
                consumers_sync();
                for (uint32_t e = tid + (hid0 - first) * CH; e < (hid1 - first) * CH; e += ATTN_CONSUMERS)
                    if (!finite16<T>(sv + vt_off<T, HD>(e / CH, e % CH))) s_bad[e / CH] = true;
                consumers_sync();
                for (uint32_t e = tid + (hid0 - first) * CH; e < (hid1 - first) * CH; e += ATTN_CONSUMERS)
                    if (s_bad[e / CH])
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(sv + vt_off<T, HD>(e / CH, e % CH)), "r"(0) : "memory");
                consumers_sync();
            }
        }

        // ---- P V ------------------------------------------------------------------------
        if constexpr (!F32) {
            if (corr[0] != 1.0f || corr[1] != 1.0f) {
#pragma unroll
                for (int n = 0; n < ND; ++n) {
                    o[n][0] *= corr[0];
                    o[n][1] *= corr[0];
                    o[n][2] *= corr[1];
                    o[n][3] *= corr[1];
                }
            }
#pragma unroll
            for (int j = 0; j < NT / 2; ++j) {
                const uint32_t pa[4] = {pf[2 * j][0], pf[2 * j][1], pf[2 * j + 1][0], pf[2 * j + 1][1]};
#pragma unroll
                for (int n = 0; n < ND / 2; ++n) {
                    uint32_t b[4];
                    ldsm4_t(sv + tile_off<T, HD>(j * 16 + (lane & 15), 2 * n + (lane >> 4)), b);
                    mma16(o[2 * n], pa, b[0], b[1], T());
                    mma16(o[2 * n + 1], pa, b[2], b[3], T());
                }
            }
        } else {
            // key 2t is column t of the product's A operand and key 2t + 1 column t + 4
            uint32_t ph[NT][4], pl[NT][4];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                split_tf32(__float_as_uint(s[j][0]), ph[j][0], pl[j][0]);
                split_tf32(__float_as_uint(s[j][2]), ph[j][1], pl[j][1]);
                split_tf32(__float_as_uint(s[j][1]), ph[j][2], pl[j][2]);
                split_tf32(__float_as_uint(s[j][3]), ph[j][3], pl[j][3]);
            }
#pragma unroll
            for (int n = 0; n < ND; ++n) {
                float hh[4] = {0.0f, 0.0f, 0.0f, 0.0f}, ll[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const uint32_t r = j * 8 + 2 * t, c = 2 * n + (g >> 2);
                    uint32_t b0, b1, h0, l0, h1, l1;
                    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(b0) : "r"(sv + v32_off<HD>(r, c) + (g & 3) * 4));
                    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(b1) : "r"(sv + v32_off<HD>(r + 1, c) + (g & 3) * 4));
                    split_tf32(b0, h0, l0);
                    split_tf32(b1, h1, l1);
                    mma8(hh, ph[j], h0, h1);
                    mma8(ll, ph[j], l0, l1);
                    mma8(ll, pl[j], h0, h1);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) o[n][i] = fmaf(o[n][i], corr[i >> 1], hh[i] + ll[i]);
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[tile % ST]);
        if (bad) {
            for (uint32_t r = hid0 - first; r < hid1 - first; ++r) {
                uint64_t off;
                if (!s_bad[r] || !attn_row(a, w, head, first + r, off)) continue;
                float p[2] = {0.0f, 0.0f};  // of vectors g and g + 8, held by the quad's lane that has column r
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (n == (int)(r >> 3) && (uint32_t)(i & 1) == (r & 1)) p[i >> 1] = s[n][i];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    p[h] = __shfl_sync(0xffffffffu, p[h], (lane & ~3u) | ((r >> 1) & 3));
                    if ((int32_t)(first + r) >= see[h]) continue;
#pragma unroll
                    for (int n = 0; n < ND; ++n)
#pragma unroll
                        for (int i = 0; i < 2; ++i) o[n][2 * h + i] = fmaf(p[h], (float)vb[off + n * 8 + 2 * t + i], o[n][2 * h + i]);
                }
            }
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
    consumers_sync();

    // ---- the outputs through shared memory, for whole rows to a thread group -----------------------
    constexpr int OP = HD + 4;
    float* s_o = reinterpret_cast<float*>(smem);  // [64][OP]
    float* s_res = s_o + ATTN_VECS * OP;          // [64][2]: (m, l)
    const uint32_t v0 = warp * 16 + g;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (t == 0) {
            s_res[(v0 + 8 * h) * 2] = m[h];
            s_res[(v0 + 8 * h) * 2 + 1] = l[h];
        }
        if (v0 + 8 * h < w.n_vec) {
#pragma unroll
            for (int n = 0; n < ND; ++n)
                *reinterpret_cast<float2*>(s_o + (v0 + 8 * h) * OP + n * 8 + 2 * t) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
        }
    }
    consumers_sync();
    pdl_wait();  // what an earlier pass left is complete

    for (uint32_t e = tid; e < w.n_vec * (HD / 4); e += ATTN_CONSUMERS) {
        const uint32_t r = e / (HD / 4), c = e % (HD / 4);
        const uint32_t i = fast_div(w.vec0 + r, a.by_group), h = head * a.group + (w.vec0 + r - i * a.group);
        const uint64_t tok = w.tok0 + i;
        const float4 x = *reinterpret_cast<const float4*>(s_o + r * OP + c * 4);
        const float L = s_res[r * 2 + 1];
        if (a.last) {
            PartSum<HD> sum;
            if (a.merge) sum.add_parts(a, tok * a.n_heads + h, c, a.merge);
            const float2 ml[1] = {make_float2(s_res[r * 2], L)};
            const float4 y[1] = {x};
            sum.template add<1>(ml, y);
            sum.template store<T>(a, tok, h, c);
        } else {
            const uint64_t at = ((uint64_t)(a.part0 + split) * a.n_tokens + tok) * a.n_heads + h;
            __stcg(reinterpret_cast<float4*>(a.part_o + at * HD) + c, x);
            if (c == 0) __stcg(a.part_ml + at, make_float2(s_res[r * 2], L));
        }
    }
}

// A thread adds the parts of four outputs of one (token, head), in part order.
template <typename T, int HD>
__global__ void __launch_bounds__(128) attn_join_kernel(const __grid_constant__ PrefixArgs a) {
    const uint64_t e = (uint64_t)blockIdx.x * 128 + threadIdx.x, stride = (uint64_t)a.n_tokens * a.n_heads;
    pdl_wait();
    pdl_trigger();
    const uint64_t id = e / (HD / 4);
    if (id >= stride) return;
    const uint32_t c = (uint32_t)(e % (HD / 4)), tok = (uint32_t)(id / a.n_heads), h = (uint32_t)(id - (uint64_t)tok * a.n_heads);
    if (a.q_start && (tok < __ldg(a.q_start) || tok >= __ldg(a.q_start + a.n_seqs))) return;  // no sequence's token
    PartSum<HD> sum;
    sum.add_parts(a, id, c, a.n_parts);
    sum.template store<T>(a, tok, h, c);
}

}  // namespace qb200
