// attn_few.cuh — the pass over paged rows for up to 32 query vectors of a KV
// head (a decoded or drafted token's group of heads).
//
// One CTA of four warps takes 16 MB vectors and a range of rows.  With so few
// vectors a row is worth little arithmetic, and what counts is how long the
// chain load -> scores -> maximum -> exponentials -> product takes for each
// warp.  So the warps share nothing until the end: each takes every fourth
// chunk of KT rows, copies them itself (16-byte cp.async into a ring of its
// own, waited for by its own copy groups), and keeps a maximum, a sum and a
// whole output of its own.  (An exchange of P between the warps, a quarter of
// the output each, saved the join at the end but took two barriers a tile: 35
// us for the own rows of 64 sequences, 8 KV heads, up to 512 rows of 128, where
// this takes 27, read cold and alone; its 67 MB are 10 us.)
//
// Rows cut into up to 8 parts are one cluster's: each CTA joins its share of
// the outputs from all CTAs' shared memory, in part order.  The prefix's
// parts (from the pass before) are added there too.
//
// Bound: bytes of K and V in the long run; at a few hundred rows a CTA the
// chain above, 3 us from a CTA's start to its first chunk, and 1 us a chunk
// and warp.  Three CTAs on an SM keep 96 to 192 KB under way.
#pragma once

#include <cooperative_groups.h>

#include "attn_prefix.cuh"

namespace qb200 {

static constexpr uint32_t FEW_THREADS = 128;

template <typename T, int HD>
struct FewShape {
    static constexpr int KT = sizeof(T) == 4 ? 8 : 16;  // rows of a chunk
    static constexpr uint32_t TILE = KT * HD * sizeof(T);
    static constexpr uint32_t STAGES = HD == 128 ? 2 : 3;
    static constexpr uint32_t RING = STAGES * 2 * TILE;  // of one warp
    static constexpr __host__ __device__ uint32_t q_bytes(int mb) { return 16 * mb * HD * sizeof(T); }
    // a warp's output takes its ring's place (or more than that)
    static constexpr __host__ __device__ uint32_t warp_bytes(int mb) {
        return RING > 16 * mb * (HD + 4) * 4u ? RING : 16 * mb * (HD + 4) * 4u;
    }
    static constexpr __host__ __device__ uint32_t smem(int mb) { return q_bytes(mb) + 4 * warp_bytes(mb); }
};

template <typename T, int HD, int MB>
__global__ void __launch_bounds__(FEW_THREADS, MB == 1 ? 3 : 2) attn_few_kernel(const __grid_constant__ PrefixArgs a) {
    namespace cg = cooperative_groups;
    constexpr bool F32 = sizeof(T) == 4;
    using S = FewShape<T, HD>;
    constexpr int KT = S::KT, ST = S::STAGES, NT = KT / 8, ND = HD / 8;
    constexpr int CH = HD * (int)sizeof(T) / 16, RP = 32 / CH, E16 = 16 / sizeof(T);
    constexpr int RV = 16 * MB, OP = HD + 4;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float2 s_ml[4][RV];   // (m, l) of each warp
    __shared__ float s_w[RV][4];     // weight of each warp's share
    __shared__ float2 s_row[RV];     // (m, l) of this CTA
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const uint32_t s_q = smem_u32(smem), s_kv = s_q + S::q_bytes(MB) + warp * S::warp_bytes(MB);
    auto warp_out = [&](uint32_t wp) { return reinterpret_cast<float*>(smem + S::q_bytes(MB) + wp * S::warp_bytes(MB)); };
    const uint32_t split = blockIdx.x, head = blockIdx.z;
    const uint32_t C = a.cluster ? gridDim.x : 1;

    if (a.first) pdl_wait();
    pdl_trigger();  // the pass after this one may start beside it
    AttnItem w;
    if (!attn_item(a, blockIdx.y, split, RV, 4 * KT, w)) {  // the same for a whole cluster
        pdl_wait();
        return;
    }
    // chunks of the CTA's rows; this warp's are warp, warp + 4, ...
    const uint32_t chunks = (w.r1 - w.r0 + KT - 1) / KT, mine = chunks > warp ? (chunks - warp + 3) / 4 : 0;
    const T* kb = reinterpret_cast<const T*>(a.k);
    const int64_t v_from_k = (const uint8_t*)a.v - (const uint8_t*)a.k;
    const uint32_t lr = lane / CH, lc = lane % CH;
    auto row_of = [&](uint32_t i) { return w.r0 + (warp + 4 * i) * KT; };
    // Places in a tile (tile_off) as a lane's part, formed once, and a step's: a step's chunk and row
    // bits are not the lane's, so they are exchanged by one XOR on the lane's part.
    constexpr uint32_t RB = HD * sizeof(T);
    constexpr bool XOR = RB >= 128;
    const uint32_t at_k = tile_off<T, HD>(lane & 7, lane >> 3), at_v = tile_off<T, HD>(lane & 15, lane >> 4), at_c = tile_off<T, HD>(lr, lc);
    auto k_at = [&](uint32_t n, uint32_t j) {  // row n * 8 + lane % 8, chunk 4 j + lane / 8
        if constexpr (XOR) return (at_k ^ ((4 * j & 7) << 4)) + (4 * j >> 3) * 128 + n * 8 * RB;
        else return tile_off<T, HD>(n * 8 + (lane & 7), 4 * j + (lane >> 3));
    };
    auto v_at = [&](uint32_t b, uint32_t j) {  // row b * 16 + lane % 16, chunk 2 j + lane / 16
        if constexpr (XOR) return (at_v ^ ((2 * j & 7) << 4)) + (2 * j >> 3) * 128 + b * 16 * RB;
        else return tile_off<T, HD>(b * 16 + (lane & 15), 2 * j + (lane >> 4));
    };
    auto c_at = [&](uint32_t p) {  // row p RP + lane / CH, chunk lane % CH
        if constexpr (XOR) return (at_c ^ ((p * RP & 7) << 4)) + p * RP * RB;
        else return tile_off<T, HD>(p * RP + lr, lc);
    };

    // The page of a chunk's rows is loaded one chunk before the copies that use it.
    uint32_t page = 0;
    auto look_up = [&](uint32_t i) {
        const uint32_t row = row_of(i) + lane;
        if (lane < KT && i < mine && row < w.r1) page = attn_page(a, w, row);
    };
    // Pages of a multiple of KT rows hold a chunk's rows one behind the other (rows begin at a multiple
    // of KT: parts do, and so does the own part without a prefix before it).
    const bool run = a.page_rows.d % KT == 0 && (w.n_prefix % KT == 0 || a.shared);
    uint32_t slot_in = 0;
    auto copy = [&](uint32_t i) {
        if (i < mine) {
            const uint32_t st = s_kv + slot_in * 2 * S::TILE, row0 = row_of(i);
            if (run && row0 + KT <= w.r1) {
                const uint64_t o = attn_offset(a, w, head, row0, __shfl_sync(0xffffffffu, page, 0));
                const uint32_t n = o == ~0ull ? 0u : 16u;
                const T* src = kb + (o == ~0ull ? 0ull : o + lr * a.row_stride) + lc * E16;
                const uint64_t by = o == ~0ull ? 0ull : RP * a.row_stride;
#pragma unroll
                for (int p = 0; p < KT / RP; ++p) {
                    cp_async16(st + c_at(p), src, n);
                    cp_async16(st + S::TILE + (F32 ? vt_off<T, HD>(p * RP + lr, lc) : c_at(p)), (const uint8_t*)src + v_from_k, n);
                    src += by;
                }
            } else {
                const uint32_t row = row0 + lane;
                const uint64_t off = lane < KT && row < w.r1 ? attn_offset(a, w, head, row, page) : ~0ull;
#pragma unroll
                for (int p = 0; p < KT / RP; ++p) {
                    const uint32_t r = p * RP + lr;
                    const uint64_t o = __shfl_sync(0xffffffffu, off, r);
                    const uint32_t n = o == ~0ull ? 0u : 16u;  // nothing read, zeros written
                    const T* src = kb + (o == ~0ull ? 0ull : o) + lc * E16;
                    cp_async16(st + tile_off<T, HD>(r, lc), src, n);
                    cp_async16(st + S::TILE + vt_off<T, HD>(r, lc), (const uint8_t*)src + v_from_k, n);
                }
            }
            slot_in = slot_in + 1 == ST ? 0 : slot_in + 1;
        }
        cp_async_commit();
    };
    look_up(0);
#pragma unroll
    for (int i = 0; i < ST - 1; ++i) {
        copy(i);
        look_up(i + 1);
    }

    // the query vectors
    for (uint32_t e = tid; e < RV * CH; e += FEW_THREADS) {
        const uint32_t r = e / CH, c = e % CH;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < w.n_vec) {
            const uint32_t i = fast_div(w.vec0 + r, a.by_group), h = head * a.group + (w.vec0 + r - i * a.group);
            v = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.q) + (uint64_t)(w.tok0 + i) * a.q_token + h * a.q_head) + c);
        }
        *reinterpret_cast<uint4*>(smem + tile_off<T, HD>(r, c)) = v;
    }
    __syncthreads();
    constexpr bool QREG = !F32 && MB == 1;  // the vectors' fragments stay in registers
    uint32_t qf[QREG ? HD / 16 : 1][4];
    if constexpr (QREG) {
#pragma unroll
        for (int j = 0; j < HD / 16; ++j) ldsm4(s_q + v_at(0, j), qf[j]);
    }

    int32_t see[MB][2];  // vectors b * 16 + g and + 8: rows that they see
    float m[MB][2], l[MB][2], o[MB][ND][4];
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            see[b][h] = w.see0 + (int32_t)fast_div(w.vec0 + b * 16 + g + 8 * h, a.by_group);
            if (!a.shared) see[b][h] = max(see[b][h], (int32_t)w.n_prefix);  // the prefix is in everyone's sight
            m[b][h] = -INFINITY;
            l[b][h] = 0.0f;
#pragma unroll
            for (int n = 0; n < ND; ++n) o[b][n][2 * h] = o[b][n][2 * h + 1] = 0.0f;
        }

    uint32_t slot = 0;
    for (uint32_t it = 0; it < mine; ++it) {
        cp_async_wait<ST - 2>();
        __syncwarp();  // this chunk is there for all lanes, and the one before it is done with
        copy(it + ST - 1);
        look_up(it + ST);
        const uint32_t sk = s_kv + slot * 2 * S::TILE, sv = sk + S::TILE;
        slot = slot + 1 == ST ? 0 : slot + 1;
        const uint32_t first = row_of(it);

        // ---- scores -----------------------------------------------------------------------
        float s[MB][NT][4];
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
            for (int n = 0; n < NT; ++n) s[b][n][0] = s[b][n][1] = s[b][n][2] = s[b][n][3] = 0.0f;
        if constexpr (!F32) {
            float s2[MB][NT][4];  // two chains of products instead of one
#pragma unroll
            for (int b = 0; b < MB; ++b)
#pragma unroll
                for (int n = 0; n < NT; ++n) s2[b][n][0] = s2[b][n][1] = s2[b][n][2] = s2[b][n][3] = 0.0f;
#pragma unroll
            for (int j = 0; j < HD / 32; ++j) {
                uint32_t q[MB][2][4];
                if constexpr (!QREG) {
#pragma unroll
                    for (int b = 0; b < MB; ++b)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            ldsm4(s_q + v_at(b, 2 * j + e), q[b][e]);
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    uint32_t k[4];
                    ldsm4(sk + k_at(n, j), k);
                    if constexpr (QREG) {
                        mma16(s[0][n], qf[2 * j], k[0], k[1], T());
                        mma16(s2[0][n], qf[2 * j + 1], k[2], k[3], T());
                    } else {
#pragma unroll
                        for (int b = 0; b < MB; ++b) {
                            mma16(s[b][n], q[b][0], k[0], k[1], T());
                            mma16(s2[b][n], q[b][1], k[2], k[3], T());
                        }
                    }
                }
            }
#pragma unroll
            for (int b = 0; b < MB; ++b)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[b][n][i] += s2[b][n][i];
        } else {
            float sl[MB][4];
#pragma unroll
            for (int b = 0; b < MB; ++b) sl[b][0] = sl[b][1] = sl[b][2] = sl[b][3] = 0.0f;
#pragma unroll 4
            for (int j = 0; j < HD / 16; ++j) {  // two k8 steps
                uint32_t k[4], kh[4], kl[4];
                ldsm4(sk + k_at(0, j), k);
#pragma unroll
                for (int i = 0; i < 4; ++i) split_tf32(k[i], kh[i], kl[i]);
#pragma unroll
                for (int b = 0; b < MB; ++b) {
                    float hh[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        uint32_t q[4], qh[4], ql[4];
                        ldsm4(s_q + v_at(b, 2 * j + e), q);
#pragma unroll
                        for (int i = 0; i < 4; ++i) split_tf32(q[i], qh[i], ql[i]);
                        mma8(hh, qh, kh[2 * e], kh[2 * e + 1]);
                        mma8(sl[b], qh, kl[2 * e], kl[2 * e + 1]);
                        mma8(sl[b], ql, kh[2 * e], kh[2 * e + 1]);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[b][0][i] += hh[i];
                }
            }
#pragma unroll
            for (int b = 0; b < MB; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[b][0][i] += sl[b][i];
        }

        // ---- mask, running maximum, exponentials ------------------------------------------
        const bool edge = first + KT > w.r1 || (int32_t)(first + KT) > w.see0;
        float corr[MB][2];
        uint32_t pf[F32 ? 1 : MB][F32 ? 1 : NT][2];
#pragma unroll
        for (int b = 0; b < MB; ++b) {
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float y = s[b][n][i] * a.c;
                    if (edge) {
                        const uint32_t row = first + n * 8 + 2 * t + (i & 1);
                        if (row >= w.r1 || (int32_t)row >= see[b][i >> 1]) y = -INFINITY;
                    }
                    s[b][n][i] = y;
                    mx[i >> 1] = fmaxf(mx[i >> 1], y);  // a NaN score goes into the sum alone
                }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
                mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
                const float M = attn_reference<T>(m[b][h], mx[h]);
                const float base = M == -INFINITY ? 0.0f : M;  // nothing seen yet: 2^-inf = 0
                corr[b][h] = M == m[b][h] ? 1.0f : ex2(m[b][h] - base);
                m[b][h] = M;
                l[b][h] *= corr[b][h];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    s[b][n][2 * h] = ex2(s[b][n][2 * h] - base);
                    s[b][n][2 * h + 1] = ex2(s[b][n][2 * h + 1] - base);
                    if constexpr (!F32) {
                        pf[b][n][h] = pack2<T>(s[b][n][2 * h], s[b][n][2 * h + 1]);
                        const float2 x = unpack2<T>(pf[b][n][h]);
                        l[b][h] += x.x + x.y;  // what is multiplied
                    } else {
                        l[b][h] += s[b][n][2 * h] + s[b][n][2 * h + 1];
                    }
                }
            }
        }

        // A row that only some of the tokens see may hold anything as far as the others are
        // concerned, and their weight 0 times an infinity or NaN in V would reach them: such
        // rows leave the chunk and are added, where seen, after the product.
        const uint32_t hid0 = max((int32_t)first, w.see0), hid1 = min(first + KT, w.r1);
        uint32_t bad = 0;  // bit r: row r of the chunk
        if (w.n_tok > 1 && !a.shared && hid0 < hid1) {
            for (uint32_t r = hid0 - first; r < hid1 - first; ++r) {
                bool ok = true;
                for (uint32_t c = lane; c < CH; c += 32) ok &= finite16<T>(sv + vt_off<T, HD>(r, c));
                if (!__all_sync(0xffffffffu, ok)) {
                    bad |= 1u << r;
                    for (uint32_t c = lane; c < CH; c += 32)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(sv + vt_off<T, HD>(r, c)), "r"(0) : "memory");
                }
            }
            __syncwarp();
        }

        // ---- P V ----------------------------------------------------------------------------
        if constexpr (!F32) {
#pragma unroll
            for (int b = 0; b < MB; ++b)
                if (corr[b][0] != 1.0f || corr[b][1] != 1.0f) {
#pragma unroll
                    for (int n = 0; n < ND; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[b][n][i] *= corr[b][i >> 1];
                }
#pragma unroll
            for (int n = 0; n < ND / 2; ++n) {
                uint32_t v[4];
                ldsm4_t(sv + v_at(0, n), v);
#pragma unroll
                for (int b = 0; b < MB; ++b) {
                    const uint32_t pa[4] = {pf[b][0][0], pf[b][0][1], pf[b][1][0], pf[b][1][1]};
                    mma16(o[b][2 * n], pa, v[0], v[1], T());
                    mma16(o[b][2 * n + 1], pa, v[2], v[3], T());
                }
            }
        } else {
            // row 2t is column t of the product's A operand and row 2t + 1 column t + 4
            uint32_t ph[MB][4], pl[MB][4];
#pragma unroll
            for (int b = 0; b < MB; ++b) {
                split_tf32(__float_as_uint(s[b][0][0]), ph[b][0], pl[b][0]);
                split_tf32(__float_as_uint(s[b][0][2]), ph[b][1], pl[b][1]);
                split_tf32(__float_as_uint(s[b][0][1]), ph[b][2], pl[b][2]);
                split_tf32(__float_as_uint(s[b][0][3]), ph[b][3], pl[b][3]);
            }
#pragma unroll
            for (int n = 0; n < ND; ++n) {
                const uint32_t c = 2 * n + (g >> 2);
                uint32_t b0, b1, h0, l0, h1, l1;
                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(b0) : "r"(sv + v32_off<HD>(2 * t, c) + (g & 3) * 4));
                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(b1) : "r"(sv + v32_off<HD>(2 * t + 1, c) + (g & 3) * 4));
                split_tf32(b0, h0, l0);
                split_tf32(b1, h1, l1);
#pragma unroll
                for (int b = 0; b < MB; ++b) {
                    float hh[4] = {0.0f, 0.0f, 0.0f, 0.0f}, ll[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    mma8(hh, ph[b], h0, h1);
                    mma8(ll, ph[b], l0, l1);
                    mma8(ll, pl[b], h0, h1);
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[b][n][i] = fmaf(o[b][n][i], corr[b][i >> 1], hh[i] + ll[i]);
                }
            }
        }
        for (; bad; bad &= bad - 1) {
            const uint32_t r = __ffs(bad) - 1;
            const T* v = reinterpret_cast<const T*>(a.v) + attn_offset(a, w, head, first + r, attn_page(a, w, first + r));
#pragma unroll
            for (int b = 0; b < MB; ++b)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float p = 0.0f;  // the quad's lane that has column r holds it
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            if ((uint32_t)n == r >> 3 && (uint32_t)i == (r & 1)) p = s[b][n][2 * h + i];
                    p = __shfl_sync(0xffffffffu, p, (lane & ~3u) | ((r >> 1) & 3));
                    if ((int32_t)(first + r) >= see[b][h]) continue;
#pragma unroll
                    for (int n = 0; n < ND; ++n)
#pragma unroll
                        for (int i = 0; i < 2; ++i) o[b][n][2 * h + i] = fmaf(p, (float)v[n * 8 + 2 * t + i], o[b][n][2 * h + i]);
                }
        }
    }
    cp_async_wait_all();
    __syncwarp();

    // ---- the warps' (m, l, o) ------------------------------------------------------------------
    float* so = warp_out(warp);
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t r = b * 16 + g + 8 * h;
            l[b][h] += __shfl_xor_sync(0xffffffffu, l[b][h], 1);
            l[b][h] += __shfl_xor_sync(0xffffffffu, l[b][h], 2);
            if (t == 0) s_ml[warp][r] = make_float2(m[b][h], l[b][h]);
            if (r < w.n_vec) {
#pragma unroll
                for (int n = 0; n < ND; ++n)
                    *reinterpret_cast<float2*>(so + r * OP + n * 8 + 2 * t) = make_float2(o[b][n][2 * h], o[b][n][2 * h + 1]);
            }
        }
    __syncthreads();
    if (tid < RV) {
        float M = -INFINITY, L = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) M = fmaxf(M, s_ml[k][tid].x);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 x = s_ml[k][tid];
            const float f = x.x == M ? 1.0f : ex2(x.x - M);
            s_w[tid][k] = f;
            L = fmaf(x.y, f, L);
        }
        s_row[tid] = make_float2(M, L);
    }
    __syncthreads();
    pdl_wait();  // what an earlier pass left is complete
    auto local = [&](uint32_t r, uint32_t c) {  // this CTA's share of four outputs
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float4 y = *reinterpret_cast<const float4*>(warp_out(k) + r * OP + c * 4);
            const float f = s_w[r][k];
            x.x = fmaf(y.x, f, x.x);
            x.y = fmaf(y.y, f, x.y);
            x.z = fmaf(y.z, f, x.z);
            x.w = fmaf(y.w, f, x.w);
        }
        return x;
    };
    cg::cluster_group cluster = cg::this_cluster();
    if (C > 1) {  // joined in place, where the cluster reads it
        for (uint32_t e = tid; e < w.n_vec * (HD / 4); e += FEW_THREADS) {
            const uint32_t r = e / (HD / 4), c = e % (HD / 4);
            const float4 x = local(r, c);
            *reinterpret_cast<float4*>(warp_out(0) + r * OP + c * 4) = x;
        }
        cluster.sync();
    }

    // ---- add the parts: every CTA of the cluster its share of the outputs --------------------------
    for (uint32_t e = (C > 1 ? split : 0) * FEW_THREADS + tid; e < w.n_vec * (HD / 4); e += FEW_THREADS * C) {
        const uint32_t r = e / (HD / 4), c = e % (HD / 4);
        const uint32_t i = fast_div(w.vec0 + r, a.by_group), h = head * a.group + (w.vec0 + r - i * a.group);
        const uint64_t tok = w.tok0 + i, id = tok * a.n_heads + h, stride = (uint64_t)a.n_tokens * a.n_heads;
        PartSum<HD> sum;
        if (a.merge) sum.add_parts(a, id, c, a.merge);
        if (C > 1) {
            float2 ml[8];
            float4 y[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const bool in = k < (int)C;
                ml[k] = in ? cluster.map_shared_rank(s_row, k)[r] : make_float2(-INFINITY, 0.0f);
                y[k] = in ? *reinterpret_cast<const float4*>(cluster.map_shared_rank(warp_out(0), k) + r * OP + c * 4)
                          : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
            sum.template add<8>(ml, y);
        } else {
            float2 ml[1] = {s_row[r]};
            float4 y[1] = {local(r, c)};
            sum.template add<1>(ml, y);
        }
        if (a.last) {
            sum.template store<T>(a, tok, h, c);
        } else {
            const uint64_t at = (uint64_t)(a.part0 + split) * stride + id;
            __stcg(reinterpret_cast<float4*>(a.part_o + at * HD) + c, sum.x);
            if (c == 0) __stcg(a.part_ml + at, make_float2(sum.M, sum.L));
        }
    }
    if (C > 1) cluster.sync();  // until the others have read this CTA's share
}

}  // namespace qb200
