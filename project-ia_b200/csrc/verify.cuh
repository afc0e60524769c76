// verify.cuh — speculative decoding's test (q_b200_verify_draft).
//
// For the drafts x_0.. of a sequence: accept while u_i q_i(x_i) < p_i(x_i);
// at the first that fails draw from r = max(p_n - q_n, 0), after the last
// accepted one from p_n.  The drawn token is the smallest index whose running
// sum of r exceeds u times the whole.
//
// A whole token hangs on these comparisons, and a running sum over 128 K
// entries has as many borders: with fp32 sums (2^-24 each) about one draw in
// forty would fall on the wrong side of one.  So r and its sums are fp64 (of
// probabilities within a lane: pairs of fp32, exact to 2^-48), and so is the
// softmax of the row that is drawn from, of weights good to 2^-37; the
// accepting tests, one border each, take their normalisers from fp32 sums.
//
// One thread-block cluster per sequence: the vocabulary is cut into one
// contiguous segment per warp of the cluster, segment sums go to every CTA
// through distributed shared memory, and the warp whose segment holds the
// border searches it (its data is still in L1/L2).  Segments are added in index
// order and lanes in a fixed one, so that equal calls give equal results; how
// the row is cut hangs on the number of sequences, and with it the sums' last
// bits.  Every row that the test needs is read from HBM once.
//
// Bound: for one sequence the dependent steps (draft id -> its probabilities
// -> the row -> the search, 6.5 us with the launch), which is why the row's
// work is spread over up to 16 CTAs, and a batch over as many as run at once.
// For a batch neither the bytes (a third of the time) nor the issue slots (37%
// busy) but the waits of the few warps that the registers leave: of a warp's
// time between two instructions a quarter goes to loads, a fifth to barriers
// and a sixth to results on their way.  64 sequences x 128256 bf16
// probabilities 18 us (33 MB, 5 us of copying), fp32 logits 48 us (66 MB, 10 us;
// an exponential in fp64 costs four fp64 operations, a series and a table
// look-up, and 64 registers spill 52 bytes; 16-bit logits spill 222 to 264).
#pragma once

#include <cooperative_groups.h>

#include "rotate.cuh"

namespace qb200 {

static constexpr uint32_t VER_THREADS = 512;
static constexpr uint32_t VER_WARPS = VER_THREADS / 32;
static constexpr uint32_t VER_MAX_CL = 16;
static constexpr uint32_t VER_MAX_DRAFT = 31;
static constexpr uint32_t VER_CHUNKS = 16;  // sums that a warp keeps of its segment's chunks, the last one of all behind

// CTAs that share an SM, and vectors of each of two rows that a lane has under
// way: probabilities take 128 registers and four vectors; logits, whose
// clusters of 8 would not all find room one CTA to an SM, half of both.
constexpr __host__ __device__ int ver_ctas(int kind) { return kind == 0 ? 1 : 2; }
constexpr __host__ __device__ int ver_vecs(int kind) { return kind == 0 ? 4 : 2; }
static constexpr int VER_SUMS = 8;  // of one row, where whole rows are summed

enum : int { VER_PROBS = 0, VER_LOGITS = 1, VER_GREEDY = 2 };

struct VerifyArgs {
    const void* target;
    const void* draft;
    uint64_t t_seq, t_row, d_seq, d_row;
    const uint32_t* draft_tokens;
    const uint32_t* draft_len;
    const float* uniform;
    uint32_t* tokens;
    uint32_t* n_tokens;
    uint32_t n_draft, vocab, seg;  // seg: entries of a warp's segment (a multiple of 8)
    uint32_t vec;                  // rows allow 16-byte accesses
    float c;                       // log2(e) / temperature
    double cd;
};

// A lane's share of NV * 32 E consecutive entries of a row from i0 on:
// 16-byte vectors of E, 32 E apart; `none` past the end.  A vector past the
// end is loaded from the row's start instead and replaced, so that all loads
// are issued before the first is looked at.
template <typename T, int E, int NV>
struct RowPart {
    Vec<T, E> v[NV];
    __device__ __forceinline__ void load(const T* row, uint32_t i0, uint32_t end, bool vec, float none) {
        const uint32_t i = i0 + (threadIdx.x & 31) * E;
        const uint32_t fill = sizeof(T) == 4 ? __float_as_uint(none) : word<T>(none, none);
        if (vec) {
#pragma unroll
            for (int k = 0; k < NV; ++k) v[k] = load_raw<T, E>(row + (i + k * 32 * E + E <= end ? i + k * 32 * E : 0u));
#pragma unroll
            for (int k = 0; k < NV; ++k)
                if (i + k * 32 * E + E > end)
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[k].w[j] = fill;
            if (i0 + NV * 32 * E <= end || end % E == 0) return;
        }
#pragma unroll
        for (int k = 0; k < NV; ++k) {  // entry by entry: rows that are not aligned, the last vector of others
            const uint32_t at = i + k * 32 * E;
            if (vec && (at + E <= end || at >= end)) continue;
            float x[E];
#pragma unroll
            for (int j = 0; j < E; ++j) x[j] = at + j < end ? (float)row[at + j] : none;
            put<E>(v[k], 0, x);
        }
    }
    template <typename U>
    static __device__ __forceinline__ uint32_t word(float a, float b) {
        if constexpr (sizeof(U) == 2) return pack2<U>(a, b);
        else return 0u;
    }
};

// 2^(d c / 1024) for -1010 < d c / 1024 <= 1 to about 1e-11: d c = k + r, a
// table of 2^(j/1024) and the series of e^(r ln 2 / 1024) to the second power
// (its argument is below 3.4e-4).  k comes out of the low word of
// d c + 1.5 * 2^52, which rounds there.
static constexpr uint32_t VER_TABLE = 1024;
__device__ __forceinline__ double exp2_table(double d, double c, const double* table) {
    const double big = 6755399441055744.0;
    const double t = fma(d, c, big), r = fma(d, c, big - t);
    const int ki = __double2loint(t);
    constexpr double c1 = 0.69314718055994530942 / VER_TABLE, c2 = c1 * c1 / 2.0;
    const double p = fma(r, fma(r, c2, c1), 1.0) * table[ki & (VER_TABLE - 1)];
    return __hiloint2double(__double2hiint(p) + ((ki >> 10) << 20), __double2loint(p));
}
// Logits up to this weigh nothing beside the maximum m: a thousand halvings
// below it, or the fp32 number next to it where one step is more than that.
__device__ __forceinline__ float logit_low(float m, float c) {
    return m < INFINITY ? fminf(m - 1000.0f / c, nextafterf(m, -INFINITY)) : m;
}
// 2^((v - m) c / 1024) for a logit v; exactly zero far below m (v <= low), and
// for NaN.  The difference comes first: v c and m c of great logits (a row
// masked with the type's lowest value) would lose it.
__device__ __forceinline__ double logit_weight(float v, float low, double c, double m, const double* table) {
    const double w = exp2_table((double)fmaxf(v, low) - m, c, table);
    return v > low ? w : 0.0;
}

// Sum of max(p - q, 0) over a lane's E entries of each of four vectors, in
// fp32 pairs (s, c) whose s + c is exact to 2^-48: the difference of p >= q
// >= 0 is hi + lo without error, and so is each addition's own error.  On
// fp64 units the two conversions of each entry alone would take 4 us for a
// batch of 64 on 128 K entries.
template <typename T, int E, int NV>
__device__ __forceinline__ double rest_sum(const RowPart<T, E, NV>& xp, const RowPart<T, E, NV>& xq, bool two) {
    static_assert(E % 2 == 0, "pairs");
    F2 s, c;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        float p[E], q[E];
        to_float(xp.v[k], p);
        if (two) to_float(xq.v[k], q);
#pragma unroll
        for (int j = 0; j < E; j += 2) {
            const float p0 = fmaxf(p[j], 0.0f), p1 = fmaxf(p[j + 1], 0.0f);  // NaN too
            F2 hi(p0, p1), lo;
            if (two) {  // q clipped into [0, p]: the difference is not below zero
                const F2 P = hi, Q(fminf(fmaxf(q[j], 0.0f), p0), fminf(fmaxf(q[j + 1], 0.0f), p1));
                hi = sub2(P, Q);
                lo = sub2(sub2(P, hi), Q);
            }
            const F2 t = add2(s, hi), z = sub2(t, s);
            const F2 err = add2(sub2(s, sub2(t, z)), sub2(hi, z));
            s = t;
            c = add2(c, err);
            if (two) c = add2(c, lo);
        }
    }
    float s0, s1, c0, c1;
    s.get(s0, s1);
    c.get(c0, c1);
    return ((double)s0 + (double)c0) + ((double)s1 + (double)c1);
}

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Order-preserving key of (value, lowest index first); 0 for NaN.  Adding
// zero makes -0 the +0 that it is equal to.
__device__ __forceinline__ unsigned long long argmax_key64(float v, uint32_t i) {
    if (!(v == v)) return 0ull;
    const uint32_t u = __float_as_uint(v + 0.0f);
    const uint32_t o = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return ((unsigned long long)o << 32) | (uint32_t)~i;
}

template <typename T, int KIND>
__global__ void __launch_bounds__(VER_THREADS, ver_ctas(KIND)) verify_kernel(const VerifyArgs a) {
    namespace cg = cooperative_groups;
    constexpr int E = 16 / sizeof(T), VER_VECS = ver_vecs(KIND);
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t CL = cluster.num_blocks(), rank = cluster.block_rank();
    const uint32_t b = blockIdx.x / CL, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t K = a.n_draft, V = a.vocab;

    constexpr uint32_t ROWS = 2 * VER_MAX_DRAFT + 2;
    __shared__ unsigned long long s_part[ROWS * VER_WARPS];       // phase A: this CTA's parts of each row
    __shared__ unsigned long long s_stat[ROWS * VER_MAX_CL];      // phase A: every CTA's share of each row
    __shared__ double s_sum[2][VER_MAX_CL * VER_WARPS];           // segment sums of target and draft
    __shared__ float s_max[VER_MAX_CL * VER_WARPS];
    __shared__ double s_rest[2][VER_MAX_CL * VER_WARPS];          // segment sums of what is drawn from
    __shared__ double s_chunk[VER_WARPS][VER_CHUNKS];             // this CTA's chunk sums
    __shared__ double s_table[KIND == VER_LOGITS ? VER_TABLE : 1];
    __shared__ float2 s_row[KIND == VER_LOGITS ? ROWS : 1];       // (maximum, sum) of each row
    __shared__ double s_z[2], s_thr;
    __shared__ float s_m[2];
    __shared__ uint32_t s_n, s_owner, s_len;

    const T* target = reinterpret_cast<const T*>(a.target) + b * a.t_seq;
    const T* draft = a.draft && KIND != VER_GREEDY ? reinterpret_cast<const T*>(a.draft) + b * a.d_seq : nullptr;
    pdl_wait();
    pdl_trigger();
    cluster.barrier_arrive();  // every CTA of the cluster runs before its shared memory is written to

    // lane i of the first warp keeps draft i
    uint32_t x = 0, len = 0;
    float u = 0.0f, pt = 0.0f, qt = 0.0f;
    bool live = false;
    if (warp == 0) {
        len = a.draft_len ? min(__ldg(a.draft_len + b), K) : K;
        if (a.draft_len && lane == 0 && rank == 0 && __ldg(a.draft_len + b) > K) qdev_fail(QDEV_BAD_ARG);
        if (lane == 0) s_len = len;
        if (lane < len) {
            x = __ldg(a.draft_tokens + (size_t)b * K + lane);
            u = __ldg(a.uniform + (size_t)b * (K + 1) + lane);
            live = x < V;
            if (live) {
                pt = (float)target[lane * a.t_row + x];
                if (draft) qt = (float)draft[lane * a.d_row + x];
            } else if (rank == 0) {
                qdev_fail(QDEV_BAD_ARG);
            }
        }
    }
    if (KIND == VER_LOGITS)
        for (uint32_t i = tid; i < VER_TABLE; i += VER_THREADS) s_table[i] = exp2((double)i / VER_TABLE);

    uint32_t Rt = 0;  // rows of the target among those that phase A sums
    // ---- phase A: what the accepting tests need of whole rows ----------------------
    if (KIND != VER_PROBS) {
        __syncthreads();
        len = s_len;
        Rt = KIND == VER_GREEDY ? len + 1 : len;
        const uint32_t R = Rt + (draft ? len : 0);
        const uint32_t P = R ? max(1u, VER_WARPS / R) : 1u;  // warps on one row
        const uint32_t share = (((V + CL - 1) / CL) + 7) & ~7u, c0 = min(rank * share, V), c1 = min(c0 + share, V);
        const uint32_t psz = (((c1 - c0 + P - 1) / P) + 7) & ~7u;
        for (uint32_t it = warp; it < R * P; it += VER_WARPS) {
            const uint32_t r = it / P, p0 = min(c0 + (it - r * P) * psz, c1), p1 = min(p0 + psz, c1);
            const T* row = r < Rt ? target + r * a.t_row : draft + (r - Rt) * a.d_row;
            if (KIND == VER_GREEDY) {
                unsigned long long best = 0;
                for (uint32_t i0 = p0; i0 < p1; i0 += VER_SUMS * 32 * E) {
                    RowPart<T, E, VER_SUMS> x;
                    x.load(row, i0, p1, a.vec, __int_as_float(0x7fffffff));
#pragma unroll
                    for (int k = 0; k < VER_SUMS; ++k) {
                        float v[E];
                        to_float(x.v[k], v);
#pragma unroll
                        for (int j = 0; j < E; ++j) {
                            const unsigned long long key = argmax_key64(v[j], i0 + (k * 32 + lane) * E + j);
                            best = key > best ? key : best;
                        }
                    }
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    const unsigned long long k = __shfl_xor_sync(0xffffffffu, best, o);
                    best = k > best ? k : best;
                }
                if (lane == 0) s_part[it] = best;
            } else {
                float m = -INFINITY, s = 0.0f;  // sum of 2^((logit - m) c)
                for (uint32_t i0 = p0; i0 < p1; i0 += VER_SUMS * 32 * E) {
                    RowPart<T, E, VER_SUMS> x;
                    x.load(row, i0, p1, a.vec, -INFINITY);
                    float mx = m, add = 0.0f;
#pragma unroll
                    for (int k = 0; k < VER_SUMS; ++k) {
                        float v[E];
                        to_float(x.v[k], v);
#pragma unroll
                        for (int j = 0; j < E; ++j) mx = fmaxf(mx, v[j]);
                    }
                    if (mx == -INFINITY) continue;
#pragma unroll
                    for (int k = 0; k < VER_SUMS; ++k) {
                        float v[E];
                        to_float(x.v[k], v);
#pragma unroll
                        for (int j = 0; j < E; ++j) add += ex2((fmaxf(v[j], -INFINITY) - mx) * a.c);  // NaN counts as zero
                    }
                    s = s * ex2((m - mx) * a.c) + add;
                    m = mx;
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
                    const float mm = fmaxf(m, m2);
                    if (mm != -INFINITY) s = s * ex2((m - mm) * a.c) + s2 * ex2((m2 - mm) * a.c);
                    m = mm;
                }
                if (lane == 0) s_part[it] = ((unsigned long long)__float_as_uint(m) << 32) | __float_as_uint(s);
            }
        }
        __syncthreads();
        cluster.barrier_wait();
        for (uint32_t e = tid; e < R * CL; e += VER_THREADS) {  // row e / CL to CTA e % CL
            const uint32_t r = e / CL, to = e - r * CL;
            unsigned long long w = s_part[r * P];
            for (uint32_t p = 1; p < P; ++p) {
                const unsigned long long w2 = s_part[r * P + p];
                if (KIND == VER_GREEDY) {
                    w = w2 > w ? w2 : w;
                } else {
                    const float m = __uint_as_float((uint32_t)(w >> 32)), m2 = __uint_as_float((uint32_t)(w2 >> 32));
                    float s = __uint_as_float((uint32_t)w);
                    const float mm = fmaxf(m, m2);
                    if (mm != -INFINITY) s = s * ex2((m - mm) * a.c) + __uint_as_float((uint32_t)w2) * ex2((m2 - mm) * a.c);
                    w = ((unsigned long long)__float_as_uint(mm) << 32) | __float_as_uint(s);
                }
            }
            *cluster.map_shared_rank(&s_stat[r * VER_MAX_CL + rank], to) = w;
        }
        cluster.sync();
        if (KIND == VER_LOGITS) {  // a lane adds a row's shares
            if (tid < R) {
                float m = -INFINITY, s = 0.0f;
                for (uint32_t k = 0; k < CL; ++k) m = fmaxf(m, __uint_as_float((uint32_t)(s_stat[tid * VER_MAX_CL + k] >> 32)));
                for (uint32_t k = 0; k < CL; ++k) {
                    const unsigned long long w = s_stat[tid * VER_MAX_CL + k];
                    const float mk = __uint_as_float((uint32_t)(w >> 32));
                    if (mk != -INFINITY) s = fmaf(__uint_as_float((uint32_t)w), ex2((mk - m) * a.c), s);
                }
                s_row[tid] = make_float2(m, s);
            }
            __syncthreads();
        }
        if (warp == 0) {
            if (KIND == VER_GREEDY) {
                unsigned long long best = 0;
                if (lane <= len)
                    for (uint32_t k = 0; k < CL; ++k) {
                        const unsigned long long w = s_stat[lane * VER_MAX_CL + k];
                        best = w > best ? w : best;
                    }
                const uint32_t top = best ? ~(uint32_t)best : 0u;
                const bool ok = lane < len && live && top == x;
                const uint32_t n = min((uint32_t)__ffs(~__ballot_sync(0xffffffffu, ok)) - 1u, len);
                const uint32_t token = __shfl_sync(0xffffffffu, top, n);
                if (rank == 0) {
                    if (lane <= K)
                        a.tokens[(size_t)b * (K + 1) + lane] = lane < n ? x : lane == n ? token : ~0u;
                    if (lane == 0) a.n_tokens[b] = n + 1;
                }
            } else {
                auto law = [&](uint32_t r, float logit) -> double {  // softmax at one entry
                    const float2 row = s_row[r];
                    const double e = exp2(((double)logit - (double)row.x) * a.cd);
                    return row.y > 0.0f && e > 0.0 ? e / (double)row.y : 0.0;
                };
                bool ok = false;
                if (live) {
                    const double p = law(lane, pt), q = draft ? law(Rt + lane, qt) : 1.0;
                    ok = (double)u * q < p;
                }
                const uint32_t n = min((uint32_t)__ffs(~__ballot_sync(0xffffffffu, ok)) - 1u, len);
                if (lane == 0) s_n = n;
            }
        }
        if (KIND == VER_GREEDY) return;
    } else if (warp == 0) {
        bool ok = false;
        if (live) {
            const double p = pt > 0.0f ? (double)pt : 0.0, q = draft ? (qt > 0.0f ? (double)qt : 0.0) : 1.0;
            ok = (double)u * q < p;
        }
        const uint32_t n = min((uint32_t)__ffs(~__ballot_sync(0xffffffffu, ok)) - 1u, len);
        if (lane == 0) s_n = n;
    }
    __syncthreads();
    const uint32_t n = s_n;
    len = s_len;

    // ---- phase B: draw from row n ----------------------------------------------------
    const T* prow = target + n * a.t_row;
    const T* qrow = draft && n < len ? draft + n * a.d_row : nullptr;
    // a draft without probabilities takes its own token out of the row
    const uint32_t gone = !draft && n < len ? __ldg(a.draft_tokens + (size_t)b * K + n) : ~0u;
    const double ct = a.cd * VER_TABLE;
    const uint32_t g = rank * VER_WARPS + warp, segs = CL * VER_WARPS;
    const uint32_t g0 = min(g * a.seg, V), g1 = min(g0 + a.seg, V);

    if (KIND == VER_LOGITS) {  // the two rows' sums, in fp64
        float m[2];
        for (int k = 0; k < 2; ++k) {  // any reference near the maximum does
            m[k] = -INFINITY;
            const uint32_t r = k ? Rt + n : n;
            if (n < len && (k == 0 || qrow)) m[k] = s_row[r].x;
        }
        if (n >= len) {  // a row that no test has looked at
            float top = -INFINITY;
            for (uint32_t i0 = g0; i0 < g1; i0 += VER_VECS * 32 * E) {
                RowPart<T, E, VER_VECS> x;
                x.load(prow, i0, g1, a.vec, -INFINITY);
#pragma unroll
                for (int k = 0; k < VER_VECS; ++k) {
                    float v[E];
                    to_float(x.v[k], v);
#pragma unroll
                    for (int j = 0; j < E; ++j) top = fmaxf(top, v[j]);
                }
            }
            top = warp_max(top);
            if (lane < CL) *cluster.map_shared_rank(&s_max[g], lane) = top;
            cluster.sync();
            for (uint32_t i = lane; i < segs; i += 32) m[0] = fmaxf(m[0], s_max[i]);
            m[0] = warp_max(m[0]);
        }
        for (int k = 0; k < 2; ++k) {
            const T* row = k ? qrow : prow;
            const double top = (double)m[k];
            const float low = logit_low(m[k], a.c);
            double s = 0.0;
            if (row && m[k] > -INFINITY && m[k] < INFINITY)
                for (uint32_t i0 = g0; i0 < g1; i0 += VER_VECS * 32 * E) {
                    RowPart<T, E, VER_VECS> x;
                    x.load(row, i0, g1, a.vec, -INFINITY);
#pragma unroll
                    for (int q = 0; q < VER_VECS; ++q) {
                        float v[E];
                        to_float(x.v[q], v);
#pragma unroll
                        for (int j = 0; j < E; ++j) s += logit_weight(v[j], low, ct, top, s_table);
                    }
                }
            s = warp_sum_f64(s);
            if (lane < CL) *cluster.map_shared_rank(&s_sum[k][g], lane) = s;
            if (tid == 0) s_m[k] = m[k];
        }
        cluster.sync();
        if (warp < 2) {
            double z = 0.0;
            for (uint32_t i = lane; i < segs; i += 32) z += s_sum[warp][i];
            z = warp_sum_f64(z);
            if (lane == 0) s_z[warp] = z > 0.0 ? 1.0 / z : 0.0;
        }
        __syncthreads();
    }
    const double mp = KIND == VER_LOGITS ? (double)s_m[0] : 0.0, mq = KIND == VER_LOGITS ? (double)s_m[1] : 0.0;
    const float lp = KIND == VER_LOGITS ? logit_low(s_m[0], a.c) : 0.0f, lq = KIND == VER_LOGITS ? logit_low(s_m[1], a.c) : 0.0f;
    const double zp = KIND == VER_LOGITS ? s_z[0] : 1.0, zq = KIND == VER_LOGITS ? s_z[1] : 1.0;
    // weights in fp64 of E entries from index i on; past the end and NaN: zero
    const float none = KIND == VER_LOGITS ? -INFINITY : 0.0f;
    auto weights = [&](const Vec<T, E>& vp, const Vec<T, E>& vq, uint32_t i, bool rest, double (&w)[E]) {
        float p[E], q[E];
        to_float(vp, p);
        const bool two = rest && qrow;
        if (two) to_float(vq, q);
#pragma unroll
        for (int j = 0; j < E; ++j) {
            double d;
            if (KIND == VER_LOGITS) {
                d = logit_weight(p[j], lp, ct, mp, s_table) * zp;
                if (two) d -= logit_weight(q[j], lq, ct, mq, s_table) * zq;
            } else {
                d = (double)p[j];
                if (two) d -= (double)fmaxf(q[j], 0.0f);  // also where q is no number
            }
            w[j] = d > 0.0 && !(rest && i + j == gone) ? d : 0.0;
        }
    };

    bool rest = n < len;
    for (int round = 0; round < 2; ++round) {
        // chunk after chunk; their sums show the search where to begin
        if (lane < VER_CHUNKS) s_chunk[warp][lane] = 0.0;
        __syncwarp();
        const bool two = rest && qrow;
        double sum = 0.0;
        for (uint32_t i0 = g0, chunk = 0; i0 < g1; i0 += VER_VECS * 32 * E, ++chunk) {
            RowPart<T, E, VER_VECS> xp, xq;
            xp.load(prow, i0, g1, a.vec, none);
            if (two) xq.load(qrow, i0, g1, a.vec, none);
            double part = 0.0;
            const bool pairs = KIND == VER_PROBS && !(rest && gone - i0 < VER_VECS * 32 * E);
            if (pairs) part = rest_sum(xp, xq, two);
            if (!pairs || !(part < INFINITY)) {  // weights near the type's largest pass fp32
                part = 0.0;
#pragma unroll
                for (int k = 0; k < VER_VECS; ++k) {
                    double w[E];
                    weights(xp.v[k], xq.v[k], i0 + (k * 32 + lane) * E, rest, w);
#pragma unroll
                    for (int j = 0; j < E; ++j) part += w[j];
                }
            }
            part = warp_sum_f64(part);
            if (lane == 0) s_chunk[warp][min(chunk, VER_CHUNKS - 1)] += part;
            sum += part;
        }
        __syncwarp();
        if (KIND == VER_PROBS && round == 0) cluster.barrier_wait();
        if (lane < CL) *cluster.map_shared_rank(&s_rest[round][g], lane) = sum;
        cluster.sync();
        if (warp == 0) {  // lane l adds segments 8l.., then the lanes in order
            double mine[VER_MAX_CL * VER_WARPS / 32], run = 0.0;
#pragma unroll
            for (int k = 0; k < (int)(VER_MAX_CL * VER_WARPS / 32); ++k) {
                const uint32_t i = lane * (VER_MAX_CL * VER_WARPS / 32) + k;
                mine[k] = i < segs ? s_rest[round][i] : 0.0;
                run += mine[k];
            }
            double incl = run;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double t = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= (uint32_t)o) incl += t;
            }
            const double total = __shfl_sync(0xffffffffu, incl, 31);
            const double thr = (double)__ldg(a.uniform + (size_t)b * (K + 1) + K) * total;
            double before = __shfl_up_sync(0xffffffffu, incl, 1);
            if (lane == 0) before = 0.0;
            uint32_t hit = ~0u, last = 0;
            double at = before, base = 0.0;
#pragma unroll
            for (int k = 0; k < (int)(VER_MAX_CL * VER_WARPS / 32); ++k) {
                const uint32_t i = lane * (VER_MAX_CL * VER_WARPS / 32) + k;
                if (mine[k] > 0.0) last = i + 1;
                if (hit == ~0u && mine[k] > 0.0 && at + mine[k] > thr) {
                    hit = i;
                    base = at;
                }
                at += mine[k];
            }
            const uint32_t vote = __ballot_sync(0xffffffffu, hit != ~0u);
            const uint32_t lasts = __reduce_max_sync(0xffffffffu, last);
            const uint32_t from = vote ? __ffs(vote) - 1 : 0;
            hit = __shfl_sync(0xffffffffu, hit, from);
            base = __shfl_sync(0xffffffffu, base, from);
            if (lane == 0) {
                // no border above thr (rounding): the last entry with weight
                s_owner = total > 0.0 ? (vote ? hit : lasts - 1) : ~0u;
                s_thr = vote ? thr - base : INFINITY;
            }
        }
        __syncthreads();
        if (s_owner != ~0u || !rest) break;
        rest = false;  // nothing is left of p - q: draw from p itself
        __syncthreads();
    }

    uint32_t token = 0;
    const bool owner = s_owner == g;
    if (owner) {
        const double thr = s_thr;
        double at = 0.0;
        uint32_t c0 = g0;
        for (uint32_t k = 0; k + 1 < VER_CHUNKS && c0 + VER_VECS * 32 * E < g1 && !(at + s_chunk[warp][k] > thr); ++k) {
            at += s_chunk[warp][k];
            c0 += VER_VECS * 32 * E;
        }
        bool found = false;
        for (uint32_t pass = 0; pass < 2 && !found; ++pass) {
            // the second pass, for a border that rounding hid: the segment's last weight
            if (pass) c0 = g0, at = -INFINITY;
            for (; c0 < g1 && !found; c0 += VER_VECS * 32 * E) {
                RowPart<T, E, VER_VECS> xp, xq;
                xp.load(prow, c0, g1, a.vec, none);
                if (rest && qrow) xq.load(qrow, c0, g1, a.vec, none);
#pragma unroll 1
                for (int k = 0; k < VER_VECS && !found; ++k) {
                    Vec<T, E> vp = xp.v[0], vq = xq.v[0];
#pragma unroll
                    for (int q = 1; q < VER_VECS; ++q)
                        if (k == q) vp = xp.v[q], vq = xq.v[q];
                    const uint32_t i = c0 + (k * 32 + lane) * E;
                    double w[E], run = 0.0;
                    weights(vp, vq, i, rest, w);
#pragma unroll
                    for (int j = 0; j < E; ++j) run += w[j];
                    double incl = run;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const double t = __shfl_up_sync(0xffffffffu, incl, o);
                        if (lane >= (uint32_t)o) incl += t;
                    }
                    const uint32_t has = __ballot_sync(0xffffffffu, run > 0.0);
                    const uint32_t vote = __ballot_sync(0xffffffffu, run > 0.0 && at + incl > thr);
                    if (has) {  // the lane with the border; without one, the last that has weight
                        const uint32_t from = vote ? __ffs(vote) - 1 : 31 - __clz(has);
                        double c = __shfl_up_sync(0xffffffffu, incl, 1);
                        c = at + (lane == 0 ? 0.0 : c);
                        uint32_t mine = 0;
                        bool met = false;
#pragma unroll
                        for (int j = 0; j < E; ++j) {
                            c += w[j];
                            if (!met && w[j] > 0.0) {
                                mine = i + j;
                                met = c > thr;
                            }
                        }
                        token = __shfl_sync(0xffffffffu, mine, from);
                        found = vote != 0;
                    }
                    at += __shfl_sync(0xffffffffu, incl, 31);
                }
            }
        }
        if (lane == 0) a.tokens[(size_t)b * (K + 1) + n] = token;
    }
    if (rank == 0 && warp == 0) {
        if (lane <= K && lane != n) a.tokens[(size_t)b * (K + 1) + lane] = lane < n ? x : ~0u;
        if (lane == n && s_owner == ~0u) a.tokens[(size_t)b * (K + 1) + n] = 0u;
        if (lane == 0) a.n_tokens[b] = n + 1;
    }
}

}  // namespace qb200
