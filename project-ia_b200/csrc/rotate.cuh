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
// Bound: bytes (3 flops for each element of 4 to 8 bytes moved), as long as
// the angles do not cost more: a sine and cosine is about 50 instructions,
// and every head of a token needs the same ones.  So a CTA takes whole tokens
// (or a run of one token's heads), forms their cosines and sines once in
// shared memory, and each thread then turns N units of E pairs (two vectors
// of E elements, 16 bytes each where alignment allows).  The N units' loads
// are issued before the angles are formed, so that they are under way
// meanwhile.  Neighbouring threads take neighbouring units of a head: every
// access is coalesced.  (Angles formed by every thread for its own unit took
// 300 instructions a unit: 70 us for 8191 x 40 x 128 bf16, where this takes 32.)
//
// Measured back to back: the 168 MB of that in 31.5 us and the 67 MB of 2048 x
// 32 x 128 fp32 in 12.5 us, 0.81 of a plain copy's rate (of a warp's time
// between two instructions a third goes to the barrier behind the angles, the
// rest to loads and results on their way); one token 3.3 to 4.4 us, the
// time of a launch.  An append of 4093 tokens (32/8 heads of 128, bf16) takes 23.6
// us, 0.65: 62 registers leave room for four CTAs on an SM, so its 2047 are 3.46
// waves, the last half empty, and every token's page and three tensors' rows are
// looked up (issue slots 41% busy).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "qorus_b200.h"

namespace qb200 {

static constexpr uint32_t ROT_THREADS = 256;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two fp32 numbers, added and multiplied side by side.
struct F2 {
    unsigned long long w;
    __device__ __forceinline__ F2() : w(0ull) {}
    __device__ __forceinline__ F2(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(w) : "f"(a), "f"(b)); }
    __device__ __forceinline__ void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(w)); }
};
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
    F2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.w) : "l"(a.w), "l"(b.w));
    return d;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.w) : "l"(a.w), "l"(b.w), "l"(c.w));
    return d;
}
__device__ __forceinline__ F2 sub2(F2 a, F2 b) {  // a - b, rounded once
    F2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.w) : "l"(b.w), "l"(F2(-1.0f, -1.0f).w), "l"(a.w));
    return d;
}

// Two 16-bit numbers in a word.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}

// E consecutive elements as they lie in memory, in 16-, 8- or single-element
// accesses; the address is aligned to min(16, E * sizeof(T)).  They are kept
// as whole words: an array of 16-bit elements is taken apart right behind its
// load, which then waits, and the loads after it with it.
template <typename T, int E>
struct Vec {
    static constexpr int WORDS = sizeof(T) * E / 4;
    uint32_t w[WORDS];
};
template <typename T>
struct Vec<T, 1> {
    T e;
};
template <typename T, int E>
__device__ __forceinline__ Vec<T, E> load_raw(const T* p) {
    Vec<T, E> v;
    if constexpr (E == 1) {
        v.e = *p;
    } else if constexpr (sizeof(T) * E >= 16) {
#pragma unroll
        for (int c = 0; c < Vec<T, E>::WORDS / 4; ++c) {
            const uint4 x = reinterpret_cast<const uint4*>(p)[c];
            v.w[4 * c] = x.x, v.w[4 * c + 1] = x.y, v.w[4 * c + 2] = x.z, v.w[4 * c + 3] = x.w;
        }
    } else {
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        v.w[0] = x.x, v.w[1] = x.y;
    }
    return v;
}
template <typename T, int E>
__device__ __forceinline__ void store_raw(T* p, const Vec<T, E>& v) {
    if constexpr (E == 1) {
        *p = v.e;
    } else if constexpr (sizeof(T) * E >= 16) {
#pragma unroll
        for (int c = 0; c < Vec<T, E>::WORDS / 4; ++c)
            reinterpret_cast<uint4*>(p)[c] = make_uint4(v.w[4 * c], v.w[4 * c + 1], v.w[4 * c + 2], v.w[4 * c + 3]);
    } else {
        *reinterpret_cast<uint2*>(p) = make_uint2(v.w[0], v.w[1]);
    }
}
// M elements from the i-th on, to fp32 and, rounded once, from fp32.
template <int M, typename T, int E>
__device__ __forceinline__ void get(const Vec<T, E>& v, int i, float (&y)[M]) {
    if constexpr (E == 1) {
        y[0] = (float)v.e;
    } else if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int k = 0; k < M / 2; ++k) {
            const float2 x = unpack2<T>(v.w[i / 2 + k]);
            y[2 * k] = x.x;
            y[2 * k + 1] = x.y;
        }
    } else {
#pragma unroll
        for (int k = 0; k < M; ++k) y[k] = __uint_as_float(v.w[i + k]);
    }
}
template <int M, typename T, int E>
__device__ __forceinline__ void put(Vec<T, E>& v, int i, const float (&y)[M]) {
    if constexpr (E == 1) {
        v.e = (T)y[0];
    } else if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int k = 0; k < M / 2; ++k) v.w[i / 2 + k] = pack2<T>(y[2 * k], y[2 * k + 1]);
    } else {
#pragma unroll
        for (int k = 0; k < M; ++k) v.w[i + k] = __float_as_uint(y[k]);
    }
}
template <typename T, int E>
__device__ __forceinline__ void to_float(const Vec<T, E>& v, float (&y)[E]) {
    get<E>(v, 0, y);
}
template <typename T, int E>
__device__ __forceinline__ void store_vec(T* p, const float (&y)[E]) {
    Vec<T, E> v;
    put<E>(v, 0, y);
    store_raw(p, v);
}
template <int M>
__device__ __forceinline__ void load_shared(const float* p, float (&y)[M]) {
    if constexpr (M == 4) {
        const float4 x = *reinterpret_cast<const float4*>(p);
        y[0] = x.x, y[1] = x.y, y[2] = x.z, y[3] = x.w;
    } else if constexpr (M == 2) {
        const float2 x = *reinterpret_cast<const float2*>(p);
        y[0] = x.x, y[1] = x.y;
    } else {
        y[0] = *p;
    }
}

// n / d for n < 2^31 by a multiplication (d fixed on the host).
struct FastDiv {
    uint32_t d, mul, shift;
};
__device__ __forceinline__ uint32_t fast_div(uint32_t n, const FastDiv& f) {
    return (__umulhi(n, f.mul) + n) >> f.shift;
}

// One kind of head in a launch: `heads` heads of every token.
struct RotateRows {
    const void* src;
    void* dst;  // the paged cache's base for keys and values
    uint32_t src_token, src_head, dst_token, dst_head;
    uint32_t heads, rotate;
};

static constexpr uint32_t ROT_ANGLES = 2048;  // cosines and sines of a CTA
static constexpr uint32_t ROT_TOKENS = 32;    // tokens of a CTA

struct RotateArgs {
    RotateRows part[3];    // append: keys, values, queries; rope: queries alone in part[2]
    const int32_t* pos;
    const int32_t* row;    // append only: < 0 is padding
    const uint32_t* seq;
    const uint32_t* pages;
    uint64_t page_stride;
    uint32_t row_stride;
    FastDiv page_rows;
    uint32_t n_pages, pages_per_seq, n_seqs;
    uint32_t n_tokens, head_dim, rot, interleaved;
    uint32_t rot_units;    // units of a row that rotate, rot / (2E); the rest is copied, E elements a unit
    uint32_t cta_tokens, cta_heads, heads;  // a CTA's share; heads of all kinds
    uint32_t row_step;     // rows that the CTA's threads take at once
    FastDiv by_units, by_heads, by_pairs;   // units of a row, cta_heads, rot / 2
    float gain, sign;
    double turns[128];
};

// One unit: pairs (a_j, b_j) in the half layout, in the interleaved one the
// pairs lie in a, then in b.  Four pairs at a time keep few numbers live.
template <typename TI, typename TO, int E>
__device__ __forceinline__ void turn_unit(const Vec<TI, E>& a, const Vec<TI, E>& b, const float* cs, const float* sn, bool inter,
                                          Vec<TO, E>& oa, Vec<TO, E>& ob) {
    constexpr int M = E >= 4 ? 4 : 1;
    if (E > 1 && inter) {
        constexpr int H = E > 1 ? E / 2 : 1;  // pairs of a, of b
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            float x[E], c[H], s[H];
            get<E>(k ? b : a, 0, x);
            load_shared<H>(cs + k * H, c);
            load_shared<H>(sn + k * H, s);
#pragma unroll
            for (int j = 0; j < H; ++j) {
                const float u = x[2 * j], v = x[2 * j + (E > 1)];
                x[2 * j] = u * c[j] - v * s[j];
                x[2 * j + (E > 1)] = u * s[j] + v * c[j];
            }
            put<E>(k ? ob : oa, 0, x);
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; i += M) {
            float x[M], y[M], c[M], s[M];
            get<M>(a, i, x);
            get<M>(b, i, y);
            load_shared<M>(cs + i, c);
            load_shared<M>(sn + i, s);
#pragma unroll
            for (int j = 0; j < M; ++j) {
                const float u = x[j], v = y[j];
                x[j] = u * c[j] - v * s[j];
                y[j] = u * s[j] + v * c[j];
            }
            put<M>(oa, i, x);
            put<M>(ob, i, y);
        }
    }
}
template <typename TI, typename TO, int E>
__device__ __forceinline__ Vec<TO, E> convert(const Vec<TI, E>& a) {
    if constexpr (std::is_same<TI, TO>::value) {
        return a;
    } else {
        Vec<TO, E> o;
        float x[E];
        get<E>(a, 0, x);
        put<E>(o, 0, x);
        return o;
    }
}

template <typename TI, typename TC, int E, int N, bool APPEND>
__global__ void __launch_bounds__(ROT_THREADS) rotate_kernel(const __grid_constant__ RotateArgs a) {
    __shared__ __align__(16) float s_cos[ROT_ANGLES], s_sin[ROT_ANGLES];
    __shared__ uint64_t s_off[ROT_TOKENS];  // append: the token's row in the cache; ~0: none
    pdl_wait();
    pdl_trigger();
    const uint32_t tid = threadIdx.x, t0 = blockIdx.x * a.cta_tokens, h0 = blockIdx.y * a.cta_heads;
    const uint32_t nt = min(a.cta_tokens, a.n_tokens - t0), nh = min(a.cta_heads, a.heads - h0);
    // this thread's unit of every row that it takes: rows rsub, rsub + step, ... of the CTA's nt x nh
    const uint32_t U = a.by_units.d, rsub = fast_div(tid, a.by_units), u = tid - rsub * U, step = a.row_step;
    const bool turn = u < a.rot_units;
    const uint32_t ia = turn ? (a.interleaved ? 2 * E * u : E * u) : a.rot + E * (u - a.rot_units);
    const uint32_t ib = a.interleaved ? ia + E : ia + a.rot / 2;
    struct Row {
        uint32_t tok, kind, head;
        bool in;
    };
    auto row_of = [&](int k) {
        Row x;
        const uint32_t r = rsub + k * step;
        x.tok = fast_div(r, a.by_heads);
        const uint32_t h = r - x.tok * a.cta_heads;
        x.in = rsub < step && x.tok < nt && h < nh;
        x.head = h0 + h;
        x.kind = 2;
        if (APPEND) {
            const uint32_t kv = a.part[0].heads;
            x.kind = x.head < kv ? 0 : x.head < 2 * kv ? 1 : 2;
            x.head -= x.kind * kv;
        }
        return x;
    };

    Vec<TI, E> va[N], vb[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const Row x = row_of(k);
        if (!x.in) continue;
        const RotateRows& p = a.part[x.kind];
        const TI* src = reinterpret_cast<const TI*>(p.src) + (uint64_t)(t0 + x.tok) * p.src_token + (uint64_t)x.head * p.src_head;
        va[k] = load_raw<TI, E>(src + ia);
        if (turn) vb[k] = load_raw<TI, E>(src + ib);
    }
    const uint32_t pairs = a.rot / 2;
    // through a generic address: every lane reads another one, which the
    // constant cache would serve one after another
    const double* turns = a.turns;
    asm volatile("" : "+l"(turns));
    for (uint32_t e = tid; e < nt * pairs; e += ROT_THREADS) {
        const uint32_t tok = fast_div(e, a.by_pairs), i = e - tok * pairs;
        const int32_t pos = __ldg((APPEND && !a.pos ? a.row : a.pos) + t0 + tok);
        double w = (double)pos * turns[i];
        w -= rint(w);
        float c, s;
        sincospif((float)(w + w), &s, &c);
        s_cos[e] = c * a.gain;
        s_sin[e] = s * a.sign;
    }
    if (APPEND && tid < nt) {
        const uint32_t t = t0 + tid;
        const int32_t row = __ldg(a.row + t);
        uint64_t off = ~0ull;
        if (row >= 0) {
            const uint32_t sq = a.seq ? __ldg(a.seq + t) : t, r = fast_div((uint32_t)row, a.page_rows);
            uint32_t pg = ~0u;
            if (sq < a.n_seqs && r < a.pages_per_seq) pg = __ldg(a.pages + (size_t)sq * a.pages_per_seq + r);
            if (pg < a.n_pages) off = pg * a.page_stride + (uint64_t)((uint32_t)row - r * a.page_rows.d) * a.row_stride;
            else qdev_fail(QDEV_BAD_ARG);
        }
        s_off[tid] = off;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const Row x = row_of(k);
        if (!x.in) continue;
        const RotateRows& p = a.part[x.kind];
        const float *cs = s_cos + x.tok * pairs + E * u, *sn = s_sin + x.tok * pairs + E * u;  // E divides both
        auto finish = [&](auto* dst, auto to) {
            using TO = decltype(to);
            Vec<TO, E> oa, ob;
            if (turn && p.rotate) {
                turn_unit<TI, TO, E>(va[k], vb[k], cs, sn, a.interleaved, oa, ob);
            } else {
                oa = convert<TI, TO, E>(va[k]);
                if (turn) ob = convert<TI, TO, E>(vb[k]);
            }
            store_raw(dst + ia, oa);
            if (turn) store_raw(dst + ib, ob);
        };
        if (APPEND) {
            const uint64_t off = s_off[x.tok];
            if (off == ~0ull) continue;  // padding, or no page
            if (x.kind < 2) {
                finish(reinterpret_cast<TC*>(p.dst) + off + (uint64_t)x.head * p.dst_head, TC());
                continue;
            }
        }
        finish(reinterpret_cast<TI*>(p.dst) + (uint64_t)(t0 + x.tok) * p.dst_token + (uint64_t)x.head * p.dst_head, TI());
    }
}

}  // namespace qb200
