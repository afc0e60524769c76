// verify.cuh — speculative decoding's test (q_b200_verify_draft).
//
// For the drafts x_0.. of a sequence: accept while u_i q_i(x_i) < p_i(x_i);
// at the first that fails draw from r = max(p_n - q_n, 0), after the last
// accepted one from p_n.  The drawn token is the smallest index whose running
// sum of r exceeds u times the whole.
//
// A whole token hangs on these comparisons, and a running sum over 128 K
// entries has as many borders: with fp32 sums (2^-24 each) about one draw in
// forty would fall on the wrong side of one.  So r and its sums are fp64, and
// so is the softmax of the row that is drawn from; the accepting tests, one
// border each, take their normalisers from fp32 sums.
//
// One thread-block cluster per sequence: the vocabulary is cut into one
// contiguous segment per warp of the cluster, segment sums go to every CTA
// through distributed shared memory, and the warp whose segment holds the
// border searches it (its data is still in L1/L2).  Sums are added in index
// order, so a result does not depend on the launch.  Every row that the test
// needs is read from HBM once.  Bound: bytes for a batch; for one sequence
// the dependent steps (draft id -> its probabilities -> the row -> the
// search), which is why the row's work is spread over up to 16 CTAs.
#pragma once

#include <cooperative_groups.h>

#include "rotate.cuh"

namespace qb200 {

static constexpr uint32_t VER_THREADS = 512;
static constexpr uint32_t VER_WARPS = VER_THREADS / 32;
static constexpr uint32_t VER_MAX_CL = 16;
static constexpr uint32_t VER_MAX_DRAFT = 31;

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

// E entries from index i of a row, `none` past its end.
template <typename T, int E>
__device__ __forceinline__ void load_row(const T* row, uint32_t i, uint32_t end, bool vec, float none, float (&v)[E]) {
    if (vec && i + E <= end) {
        to_float(load_raw<T, E>(row + i), v);
    } else {
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] = i + j < end ? (float)row[i + j] : none;
    }
}

// 2^y for y <= 0 to about 1e-13: y = k/256 + r, a table of 2^(j/256) and the
// series of e^(r ln 2) to the third power (|r ln 2| < 1.4e-3).
__device__ __forceinline__ double exp2_table(double y, const double* table) {
    if (!(y > -1000.0)) return 0.0;
    const double k = rint(y * 256.0);
    const double r = fma(k, -1.0 / 256.0, y) * 0.69314718055994530942;
    const int ki = (int)k;
    const double p = fma(r, fma(r, fma(r, 1.0 / 6.0, 0.5), 1.0), 1.0) * table[ki & 255];
    return __hiloint2double(__double2hiint(p) + ((ki >> 8) << 20), __double2loint(p));
}

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Order-preserving key of (value, lowest index first); 0 for NaN.
__device__ __forceinline__ unsigned long long argmax_key64(float v, uint32_t i) {
    if (!(v == v)) return 0ull;
    const uint32_t u = __float_as_uint(v);
    const uint32_t o = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return ((unsigned long long)o << 32) | (uint32_t)~i;
}

template <typename T, int KIND>
__global__ void __launch_bounds__(VER_THREADS) verify_kernel(const VerifyArgs a) {
    namespace cg = cooperative_groups;
    constexpr int E = 16 / sizeof(T);
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t CL = cluster.num_blocks(), rank = cluster.block_rank();
    const uint32_t b = blockIdx.x / CL, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t K = a.n_draft, V = a.vocab;

    constexpr uint32_t ROWS = 2 * VER_MAX_DRAFT + 2;
    __shared__ unsigned long long s_part[ROWS * VER_WARPS];       // phase A: this CTA's parts of each row
    __shared__ unsigned long long s_stat[ROWS * VER_MAX_CL];      // phase A: every CTA's share of each row
    __shared__ double s_sum[2][VER_MAX_CL * VER_WARPS];           // segment sums of target and draft
    __shared__ float s_max[2][VER_MAX_CL * VER_WARPS];
    __shared__ double s_rest[2][VER_MAX_CL * VER_WARPS];          // segment sums of what is drawn from
    __shared__ double s_table[256];
    __shared__ double s_z[2], s_thr;
    __shared__ float s_m[2];
    __shared__ uint32_t s_n, s_owner, s_len;

    const T* target = reinterpret_cast<const T*>(a.target) + b * a.t_seq;
    const T* draft = a.draft && KIND != VER_GREEDY ? reinterpret_cast<const T*>(a.draft) + b * a.d_seq : nullptr;
    cluster.sync();  // every CTA of the cluster runs before its shared memory is written to

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
        if (tid < 256) s_table[tid] = exp2((double)tid / 256.0);

    // ---- phase A: what the accepting tests need of whole rows ----------------------
    if (KIND != VER_PROBS) {
        __syncthreads();
        len = s_len;
        const uint32_t Rt = KIND == VER_GREEDY ? len + 1 : len, R = Rt + (draft ? len : 0);
        const uint32_t P = R ? max(1u, VER_WARPS / R) : 1u;  // warps on one row
        const uint32_t share = (((V + CL - 1) / CL) + 7) & ~7u, c0 = min(rank * share, V), c1 = min(c0 + share, V);
        const uint32_t psz = (((c1 - c0 + P - 1) / P) + 7) & ~7u;
        for (uint32_t it = warp; it < R * P; it += VER_WARPS) {
            const uint32_t r = it / P, p0 = min(c0 + (it - r * P) * psz, c1), p1 = min(p0 + psz, c1);
            const T* row = r < Rt ? target + r * a.t_row : draft + (r - Rt) * a.d_row;
            if (KIND == VER_GREEDY) {
                unsigned long long best = 0;
                for (uint32_t i = p0 + lane * E; i < p1; i += 32 * E) {
                    float v[E];
                    load_row<T, E>(row, i, p1, a.vec, __int_as_float(0x7fffffff), v);
#pragma unroll
                    for (int j = 0; j < E; ++j) {
                        const unsigned long long k = argmax_key64(v[j], i + j);
                        best = k > best ? k : best;
                    }
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    const unsigned long long k = __shfl_xor_sync(0xffffffffu, best, o);
                    best = k > best ? k : best;
                }
                if (lane == 0) s_part[it] = best;
            } else {
                float m = -INFINITY, s = 0.0f;  // of y = logit * c, the softmax in powers of two
                for (uint32_t i = p0 + lane * E; i < p1; i += 32 * E) {
                    float v[E], mx = m;
                    load_row<T, E>(row, i, p1, a.vec, -INFINITY, v);
#pragma unroll
                    for (int j = 0; j < E; ++j) {
                        v[j] *= a.c;
                        mx = fmaxf(mx, v[j]);
                    }
                    if (mx == -INFINITY) continue;
                    float add = 0.0f;
#pragma unroll
                    for (int j = 0; j < E; ++j) {
                        const float e = exp2f(v[j] - mx);
                        add += e > 0.0f ? e : 0.0f;  // NaN counts as zero
                    }
                    s = s * exp2f(m - mx) + add;
                    m = mx;
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
                    const float mm = fmaxf(m, m2);
                    if (mm != -INFINITY) s = s * exp2f(m - mm) + s2 * exp2f(m2 - mm);
                    m = mm;
                }
                if (lane == 0) s_part[it] = ((unsigned long long)__float_as_uint(m) << 32) | __float_as_uint(s);
            }
        }
        __syncthreads();
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
                    if (mm != -INFINITY) s = s * exp2f(m - mm) + __uint_as_float((uint32_t)w2) * exp2f(m2 - mm);
                    w = ((unsigned long long)__float_as_uint(mm) << 32) | __float_as_uint(s);
                }
            }
            *cluster.map_shared_rank(&s_stat[r * VER_MAX_CL + rank], to) = w;
        }
        cluster.sync();
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
                    float m = -INFINITY;
                    for (uint32_t k = 0; k < CL; ++k)
                        m = fmaxf(m, __uint_as_float((uint32_t)(s_stat[r * VER_MAX_CL + k] >> 32)));
                    double s = 0.0;
                    for (uint32_t k = 0; k < CL; ++k) {
                        const unsigned long long w = s_stat[r * VER_MAX_CL + k];
                        const float mk = __uint_as_float((uint32_t)(w >> 32));
                        if (mk != -INFINITY) s += (double)__uint_as_float((uint32_t)w) * (double)exp2f(mk - m);
                    }
                    const double e = exp2((double)logit * a.cd - (double)m);
                    return s > 0.0 && e > 0.0 ? e / s : 0.0;
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
    const uint32_t g = rank * VER_WARPS + warp, segs = CL * VER_WARPS;
    const uint32_t g0 = min(g * a.seg, V), g1 = min(g0 + a.seg, V);

    if (KIND == VER_LOGITS) {  // the two rows' maxima and sums, in fp64
        for (int k = 0; k < 2; ++k) {
            const T* row = k ? qrow : prow;
            float m = -INFINITY;
            double s = 0.0;
            if (row) {
                for (uint32_t i = g0 + lane * E; i < g1; i += 32 * E) {
                    float v[E];
                    load_row<T, E>(row, i, g1, a.vec, -INFINITY, v);
#pragma unroll
                    for (int j = 0; j < E; ++j) m = fmaxf(m, v[j]);
                }
                m = warp_max(m);
                if (m > -INFINITY && m < INFINITY)
                    for (uint32_t i = g0 + lane * E; i < g1; i += 32 * E) {
                        float v[E];
                        load_row<T, E>(row, i, g1, a.vec, -INFINITY, v);
#pragma unroll
                        for (int j = 0; j < E; ++j) s += exp2_table(((double)v[j] - (double)m) * a.cd, s_table);
                    }
                s = warp_sum_f64(s);
            }
            if (lane < CL) {
                *cluster.map_shared_rank(&s_max[k][g], lane) = m;
                *cluster.map_shared_rank(&s_sum[k][g], lane) = s;
            }
        }
        cluster.sync();
        if (warp < 2) {
            float m = -INFINITY;
            for (uint32_t i = lane; i < segs; i += 32) m = fmaxf(m, s_max[warp][i]);
            m = warp_max(m);
            double z = 0.0;
            for (uint32_t i = lane; i < segs; i += 32)
                z += s_sum[warp][i] * exp2_table(((double)s_max[warp][i] - (double)m) * a.cd, s_table);
            z = warp_sum_f64(z);
            if (lane == 0) {
                s_m[warp] = m;
                s_z[warp] = z > 0.0 ? 1.0 / z : 0.0;
            }
        }
        __syncthreads();
    }
    const double mp = KIND == VER_LOGITS ? (double)s_m[0] : 0.0, mq = KIND == VER_LOGITS ? (double)s_m[1] : 0.0;
    const double zp = KIND == VER_LOGITS ? s_z[0] : 1.0, zq = KIND == VER_LOGITS ? s_z[1] : 1.0;
    // weights of entries i.. in fp64; past the end and NaN: zero
    auto weights = [&](uint32_t i, bool rest, double (&w)[E]) {
        float p[E], q[E];
        load_row<T, E>(prow, i, g1, a.vec, KIND == VER_LOGITS ? -INFINITY : 0.0f, p);
        const bool two = rest && qrow;
        if (two) load_row<T, E>(qrow, i, g1, a.vec, KIND == VER_LOGITS ? -INFINITY : 0.0f, q);
#pragma unroll
        for (int j = 0; j < E; ++j) {
            double d;
            if (KIND == VER_LOGITS) {
                d = exp2_table(((double)p[j] - mp) * a.cd, s_table) * zp;
                if (two) d -= exp2_table(((double)q[j] - mq) * a.cd, s_table) * zq;
            } else {
                d = (double)p[j];
                if (two && q[j] > 0.0f) d -= (double)q[j];
            }
            w[j] = d > 0.0 && !(rest && i + j == gone) ? d : 0.0;
        }
    };

    bool rest = n < len;
    for (int round = 0; round < 2; ++round) {
        double sum = 0.0;
        for (uint32_t i = g0 + lane * E; i < g1; i += 32 * E) {
            double w[E];
            weights(i, rest, w);
#pragma unroll
            for (int j = 0; j < E; ++j) sum += w[j];
        }
        sum = warp_sum_f64(sum);
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
        bool found = false;
        for (uint32_t i0 = g0; i0 < g1 && !found; i0 += 32 * E) {
            double w[E], run = 0.0;
            weights(i0 + lane * E, rest, w);
            uint32_t last = 0;
#pragma unroll
            for (int j = 0; j < E; ++j) {
                run += w[j];
                if (w[j] > 0.0) last = i0 + lane * E + j + 1;
            }
            double incl = run;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double t = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= (uint32_t)o) incl += t;
            }
            double before = __shfl_up_sync(0xffffffffu, incl, 1);
            if (lane == 0) before = 0.0;
            const uint32_t vote = __ballot_sync(0xffffffffu, run > 0.0 && at + incl > thr);
            const uint32_t lasts = __reduce_max_sync(0xffffffffu, last);
            if (lasts) token = lasts - 1;  // stays where no border is met
            if (vote) {
                const uint32_t from = __ffs(vote) - 1;
                uint32_t mine = last ? last - 1 : 0;
                double c = at + before;
                bool met = false;
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    c += w[j];
                    if (!met && w[j] > 0.0 && c > thr) {
                        mine = i0 + lane * E + j;
                        met = true;
                    }
                }
                token = __shfl_sync(0xffffffffu, mine, from);
                found = true;
            }
            at += __shfl_sync(0xffffffffu, incl, 31);
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
