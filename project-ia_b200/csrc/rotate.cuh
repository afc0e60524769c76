// rotate.cuh — rotary positions (q_b200_rope) and the paged append that
// rotates on the way (q_b200_kv_append).
//
// A pair (a, b) of a row turns by its position's angle:
//   a' = a cos - b sin,  b' = a sin + b cos,  angle = pos * f_i.
// The angle is kept in turns, t = pos * (f_i / 2 pi), formed in 64 bits and
// reduced to its fraction before it is rounded to fp32: an fp32 product
// would be off by pos * 2^-24 radians (0.06 at a million).  sincospif takes
// the fraction in half turns, so nothing else is reduced.  Products and the
// rotation are fp32; each output is rounded once to its type.
//
// Bound: bytes (3 flops for each element of 4 to 8 bytes moved).  One thread
// takes one unit (E pairs: two vectors of E elements, E sized to 16-byte
// accesses of the narrower type, or one pair where alignment allows no more)
// of HB consecutive heads of one token: its cosines are computed once for
// the HB heads, and the HB * 2 loads are in flight together.  Neighbouring
// threads take neighbouring units of the same head, so every access is
// coalesced.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "qorus_b200.h"

namespace qb200 {

static constexpr uint32_t ROT_THREADS = 256;

// E consecutive elements to and from fp32; 4-, 8-, 16- or 32-byte accesses,
// the address aligned to min(16, E * sizeof(T)).
template <typename T, int E>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[E]) {
    if constexpr (sizeof(T) * E >= 16) {
#pragma unroll
        for (int c = 0; c < (int)sizeof(T) * E / 16; ++c) {
            const uint4 w = reinterpret_cast<const uint4*>(p)[c];
            const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
            for (int i = 0; i < 16 / (int)sizeof(T); ++i) v[c * (16 / sizeof(T)) + i] = (float)e[i];
        }
    } else if constexpr (sizeof(T) * E == 8) {
        const uint2 w = *reinterpret_cast<const uint2*>(p);
        const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = (float)e[i];
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = (float)p[i];
    }
}

template <typename T, int E>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[E]) {
    if constexpr (sizeof(T) * E >= 16) {
#pragma unroll
        for (int c = 0; c < (int)sizeof(T) * E / 16; ++c) {
            uint4 w;
            T* e = reinterpret_cast<T*>(&w);
#pragma unroll
            for (int i = 0; i < 16 / (int)sizeof(T); ++i) e[i] = (T)v[c * (16 / sizeof(T)) + i];
            reinterpret_cast<uint4*>(p)[c] = w;
        }
    } else if constexpr (sizeof(T) * E == 8) {
        uint2 w;
        T* e = reinterpret_cast<T*>(&w);
#pragma unroll
        for (int i = 0; i < E; ++i) e[i] = (T)v[i];
        *reinterpret_cast<uint2*>(p) = w;
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) p[i] = (T)v[i];
    }
}

// n / d for n < 2^31 by a multiplication (d fixed on the host).
struct FastDiv {
    uint32_t d, mul, shift;
};
__device__ __forceinline__ uint32_t fast_div(uint32_t n, const FastDiv& f) {
    return (__umulhi(n, f.mul) + n) >> f.shift;
}

// One kind of head in a launch: rows of `heads` heads of every token.
struct RotateRows {
    const void* src;
    void* dst;  // the paged cache's base for keys and values
    uint64_t src_token, src_head, dst_token, dst_head;
    uint32_t heads, chunks;  // chunks of HB heads
    uint32_t rotate, paged;
};

struct RotateArgs {
    RotateRows part[3];    // append: keys, values, queries; rope: queries alone in part[2]
    const int32_t* pos;
    const int32_t* row;    // append only: < 0 is padding
    const uint32_t* seq;
    const uint32_t* pages;
    uint64_t page_stride, row_stride;
    FastDiv page_rows;
    uint32_t n_pages, pages_per_seq, n_seqs;
    uint32_t n_tokens, head_dim, rot, interleaved;
    uint32_t units;        // units of a row: rot / (2E) rotating, the rest copied
    uint32_t rot_units;
    FastDiv by_units, by_chunks;
    uint64_t n_items;      // threads with work: n_tokens * chunks * units
    float gain, sign;
    double turns[128];
};

template <typename TI, typename TO, int E, int HB>
__device__ __forceinline__ void rotate_heads(const TI* src, uint64_t src_head, TO* dst, uint64_t dst_head, uint32_t n,
                                             uint32_t ia, uint32_t ib, bool rot, bool inter, const float (&cs)[E],
                                             const float (&sn)[E]) {
    float a[HB][E], b[HB][E];
#pragma unroll
    for (int h = 0; h < HB; ++h)
        if (h < (int)n) {
            load_vec<TI, E>(src + h * src_head + ia, a[h]);
            if (ib != ~0u) load_vec<TI, E>(src + h * src_head + ib, b[h]);
        }
#pragma unroll
    for (int h = 0; h < HB; ++h) {
        if (h >= (int)n) break;
        if (rot) {
            if (inter && E > 1) {  // (a0 a1)(a2 a3)... (b0 b1)...: pair j in elements 2j, 2j+1 of a then b
#pragma unroll
                for (int j = 0; j < E / 2; ++j) {
                    const float x0 = a[h][2 * j], x1 = a[h][2 * j + 1], y0 = b[h][2 * j], y1 = b[h][2 * j + 1];
                    a[h][2 * j] = x0 * cs[j] - x1 * sn[j];
                    a[h][2 * j + 1] = x0 * sn[j] + x1 * cs[j];
                    b[h][2 * j] = y0 * cs[E / 2 + j] - y1 * sn[E / 2 + j];
                    b[h][2 * j + 1] = y0 * sn[E / 2 + j] + y1 * cs[E / 2 + j];
                }
            } else {
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    const float x = a[h][j], y = b[h][j];
                    a[h][j] = x * cs[j] - y * sn[j];
                    b[h][j] = x * sn[j] + y * cs[j];
                }
            }
        }
        store_vec<TO, E>(dst + h * dst_head + ia, a[h]);
        if (ib != ~0u) store_vec<TO, E>(dst + h * dst_head + ib, b[h]);
    }
}

template <typename TI, typename TC, int E, int HB>
__global__ void __launch_bounds__(ROT_THREADS) rotate_kernel(const __grid_constant__ RotateArgs a) {
    __shared__ double s_turns[128];
    if (threadIdx.x < a.rot / 2) s_turns[threadIdx.x] = a.turns[threadIdx.x];
    __syncthreads();
    const uint64_t id = (uint64_t)blockIdx.x * ROT_THREADS + threadIdx.x;
    if (id >= a.n_items) return;
    const uint32_t n = (uint32_t)id;
    const uint32_t rc = fast_div(n, a.by_units), u = n - rc * a.by_units.d;
    const uint32_t t = fast_div(rc, a.by_chunks);
    uint32_t c = rc - t * a.by_chunks.d;
    int kind = 0;
    while (kind < 2 && c >= a.part[kind].chunks) c -= a.part[kind++].chunks;
    const RotateRows& p = a.part[kind];
    uint64_t cache_off = 0;
    int32_t pos;
    if (a.row) {
        const int32_t row = __ldg(a.row + t);
        if (row < 0) return;
        pos = a.pos ? __ldg(a.pos + t) : row;
        if (p.paged) {
            const uint32_t sq = a.seq ? __ldg(a.seq + t) : t, r = fast_div((uint32_t)row, a.page_rows);
            uint32_t pg = ~0u;
            if (sq < a.n_seqs && r < a.pages_per_seq) pg = __ldg(a.pages + (size_t)sq * a.pages_per_seq + r);
            if (pg >= a.n_pages) {
                qdev_fail(QDEV_BAD_ARG);
                return;
            }
            cache_off = pg * a.page_stride + (uint64_t)((uint32_t)row - r * a.page_rows.d) * a.row_stride;
        }
    } else {
        pos = __ldg(a.pos + t);
    }
    const bool turning = u < a.rot_units;
    const bool rot = p.rotate && turning;
    uint32_t ia, ib;
    if (turning) {
        ia = a.interleaved ? 2 * E * u : E * u;
        ib = a.interleaved ? ia + E : ia + a.rot / 2;
    } else {
        ia = a.rot + E * (u - a.rot_units);
        ib = ~0u;
    }
    float cs[E], sn[E];
    if (rot) {
#pragma unroll
        for (int j = 0; j < E; ++j) {
            double w = (double)pos * s_turns[E * u + j];
            w -= rint(w);
            sincospif((float)(w + w), &sn[j], &cs[j]);
            cs[j] *= a.gain;
            sn[j] *= a.sign;
        }
    }
    const uint32_t h0 = c * HB, nh = min((uint32_t)HB, p.heads - h0);
    const TI* src = reinterpret_cast<const TI*>(p.src) + t * p.src_token + h0 * p.src_head;
    if (p.paged)
        rotate_heads<TI, TC, E, HB>(src, p.src_head, reinterpret_cast<TC*>(p.dst) + cache_off + h0 * p.dst_head,
                                    p.dst_head, nh, ia, ib, rot, a.interleaved, cs, sn);
    else
        rotate_heads<TI, TI, E, HB>(src, p.src_head, reinterpret_cast<TI*>(p.dst) + t * p.dst_token + h0 * p.dst_head,
                                    p.dst_head, nh, ia, ib, rot, a.interleaved, cs, sn);
}

}  // namespace qb200
