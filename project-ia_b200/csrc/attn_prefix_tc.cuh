// attn_prefix_tc.cuh — the shared prefix's pass on tcgen05 (fp16 and bf16
// caches, head_dim 64 or 128).
//
// All new tokens' query vectors of a KV head (tokens x G heads) meet the same
// rows, so the pass is a matrix product: S = Q K^T and O += P V with 128
// query vectors as the MMA's M, 128 rows of the cache as one tile.  One CTA
// runs two streams, each with scores and an output of its own in TMEM
// (columns [0,128) and [128,256): S0, S1; [256,..) and [384,..): O0, O1):
//   two tiles of vectors, the same rows (more than 128 vectors), or
//   one tile of vectors, even and odd row tiles (up to 128),
// so that one stream's products run while the other's exponentials do.
//
// Roles: warps 0-3 and 4-7 are the streams' softmax, a thread per vector
// (its row of S lies in its own TMEM lane, so maximum and sum need no
// exchange); warps 8-11 copy rows of K and V (16-byte cp.async into the
// 128-byte swizzle that the MMA's descriptors name; a row's page is looked up
// by one lane); one lane of warp 12 issues the MMAs.  P overwrites S in TMEM
// in 16 bits (the operand type) and is the A operand of P V from there; V is
// used as it lies in the cache, [row][dim], as an MN-major B operand.
//
// The running maximum moves only when a row tile exceeds it by 2^8: then the
// output is rescaled in TMEM; until then exponentials may reach 256, which
// fp16 holds, and the quotient o / l is the same.
//
// Bound: for up to 128 vectors the bytes of K and V; beyond, the tensor pipe
// (4 x 128 x 128 x head_dim flops a tile) beside the exponentials (128 x 128
// of them a tile on 16 lanes of the special function unit: as long as the
// products at head_dim 128).
#pragma once

#include "attn_prefix.cuh"
#include "prefill.cuh"

namespace qb200 {

static constexpr uint32_t TC_THREADS = 416;
static constexpr uint32_t TC_ROWS = 128;

template <int HD>
struct TcShape {
    static constexpr uint32_t SLOTS = HD == 128 ? 5 : 9;        // K and V tiles in the ring
    static constexpr uint32_t TILE = TC_ROWS * HD * 2;          // one K or V tile, one tile of Q
    static constexpr uint32_t PANEL = TC_ROWS * 128;            // 64 columns of it
    static constexpr size_t SMEM = (size_t)(2 + SLOTS) * TILE + 1024 + 256;
};

// Descriptor of an MN-major operand in the 128-byte swizzle: 64 contiguous
// elements x 8 rows make 1024 bytes, row groups follow each other (SBO), the
// next 64 elements are a panel away (LBO).
__device__ __forceinline__ uint64_t umma_desc_sw128_mn(uint32_t saddr, uint32_t panel) {
    uint64_t d = (uint64_t)((saddr & 0x3FFFFu) >> 4);
    d |= (uint64_t)(panel >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

// A from TMEM.
__device__ __forceinline__ void umma_f16_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t b, uint32_t acc, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b), "r"(idesc), "r"(acc));
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}

template <typename T, int HD>
__global__ void __launch_bounds__(TC_THREADS, 1) attn_prefix_tc_kernel(const __grid_constant__ PrefixArgs a) {
    using S = TcShape<HD>;
    constexpr uint32_t NS = S::SLOTS, CH = HD / 8;
    constexpr uint32_t FMT = std::is_same<T, __half>::value ? 0u : 1u;
    // D fp32; A and B of the cache's type; K-major A; N and M in the upper fields
    constexpr uint32_t ID_QK = (1u << 4) | (FMT << 7) | (FMT << 10) | ((TC_ROWS >> 3) << 17) | ((128u >> 4) << 24);
    constexpr uint32_t ID_PV = (1u << 4) | (FMT << 7) | (FMT << 10) | (1u << 16) | ((HD >> 3) << 17) | ((128u >> 4) << 24);
    extern __shared__ uint8_t tc_smem_raw[];
    const uint32_t base = (smem_u32(tc_smem_raw) + 1023u) & ~1023u;
    uint8_t* smem = tc_smem_raw + (base - smem_u32(tc_smem_raw));
    const uint32_t s_q = base, s_kv = base + 2 * S::TILE;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + (2 + NS) * S::TILE);
    uint64_t* empty = full + NS;
    uint64_t* s_full = empty + NS;  // a stream's scores are there
    uint64_t* p_full = s_full + 2;  // its exponentials are
    uint64_t* o_full = p_full + 2;  // its output is complete
    uint64_t* q_full = o_full + 2;
    uint64_t* drain = q_full + 1;   // every product is done
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);

    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, head = blockIdx.z, split = blockIdx.x;
    pdl_trigger();  // the pass over the own rows may start beside this one
    const bool pair = !a.alternate;  // two tiles of vectors

    AttnItem w;
    const bool any = attn_item(a, blockIdx.y, split, pair ? 256 : 128, TC_ROWS, w);
    const uint32_t n_tiles = any ? (w.r1 - w.r0 + TC_ROWS - 1) / TC_ROWS : 0;
    if (tid == 0) {
        for (uint32_t i = 0; i < NS; ++i) {
            mbar_init(&full[i], 4);
            mbar_init(&empty[i], 1);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(&s_full[t], 1);
            mbar_init(&p_full[t], 4);
            mbar_init(&o_full[t], 1);
        }
        mbar_init(q_full, 8);
        mbar_init(drain, 1);
        fence_mbar_init();
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp < 8) {
        // ---- softmax ----------------------------------------------------------------------
        const uint32_t t = warp >> 2, row = tid & 127;
        const uint32_t lanes = tmem + (((warp & 3) * 32u) << 16), ts = lanes + t * 128, to = lanes + 256 + t * 128;
        {  // Q, one tile a stream, or the one tile by halves
            const uint32_t nv = any ? w.n_vec : 0, v0 = pair ? t * 128 : 0, r0 = pair ? 0 : t * 64, r1 = pair ? 128 : r0 + 64;
            const uint32_t dst = s_q + (pair ? t * S::TILE : 0);
            for (uint32_t e = row; e < (r1 - r0) * CH; e += 128) {
                const uint32_t r = r0 + e / CH, c = e % CH, v = v0 + r;
                uint4 x = make_uint4(0, 0, 0, 0);
                if (v < nv) {
                    const uint32_t i = fast_div(w.vec0 + v, a.by_group), h = head * a.group + (w.vec0 + v - i * a.group);
                    x = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.q) + (uint64_t)i * a.q_token + h * a.q_head) + c);
                }
                const uint32_t at = dst + (c >> 3) * S::PANEL + r * 128 + (((c & 7) ^ (r & 7)) << 4);
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
        }
        const uint32_t mine = pair ? n_tiles : (n_tiles + 1 - t) / 2;
        float m = -INFINITY, l = 0.0f;
        bool alive = true;
        for (uint32_t j = 0; j < mine && alive; ++j) {
            const uint32_t tile = pair ? j : 2 * j + t;
            alive = __all_sync(0xffffffffu, mbar_wait(&s_full[t], j & 1, QDEV_WAIT_FULL_TIMEOUT));
            if (!alive) break;
            tc_fence_after();
            const uint32_t cols = min(TC_ROWS, w.r1 - w.r0 - tile * TC_ROWS);  // rows past the end score nothing
            float mx = -INFINITY;
#pragma unroll
            for (uint32_t c = 0; c < 4; ++c) {
                float v[32];
                tmem_ld32(ts + c * 32, v);
                if (cols < TC_ROWS) {
#pragma unroll
                    for (uint32_t i = 0; i < 32; ++i)
                        if (c * 32 + i >= cols) v[i] = -INFINITY;
                }
#pragma unroll
                for (int i = 0; i < 32; ++i) mx = fmaxf(mx, v[i]);
            }
            mx *= a.c;  // c > 0
            const bool move = mx > m + 8.0f;  // also from -infinity
            if (__any_sync(0xffffffffu, move)) {
                const float f = move ? (m == -INFINITY ? 0.0f : ex2(m - mx)) : 1.0f;
                if (move) {
                    m = mx;
                    l *= f;
                }
                if (j > 0) {
#pragma unroll 1
                    for (uint32_t c = 0; c < HD / 32; ++c) {
                        float v[32];
                        tmem_ld32(to + c * 32, v);
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] *= f;
                        tmem_st32(to + c * 32, v);
                    }
                }
            }
            const float sub = m == -INFINITY ? 0.0f : -m;
#pragma unroll
            for (uint32_t c = 0; c < 4; ++c) {
                float v[32];
                tmem_ld32(ts + c * 32, v);
                uint32_t p[16];
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    v[i] = ex2(fmaf(v[i], a.c, sub));
                    if (cols < TC_ROWS && c * 32 + i >= cols) v[i] = 0.0f;
                    l += v[i];
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) p[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
                tmem_st16(ts + c * 16, p);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[t]);
        }
        // ---- this stream's part ----
        bool ok = alive;
        if (mine && alive) ok = __all_sync(0xffffffffu, mbar_wait(&o_full[t], 0, QDEV_WAIT_FULL_TIMEOUT));
        tc_fence_after();
        const uint32_t v = (pair ? t * 128 : 0) + row;
        const bool valid = any && v < w.n_vec;
        uint64_t at = 0;
        if (valid) {
            const uint32_t i = fast_div(w.vec0 + v, a.by_group), h = head * a.group + (w.vec0 + v - i * a.group);
            const uint32_t part = pair ? split : 2 * split + t;
            at = ((uint64_t)part * a.n_tokens + i) * a.n_heads + h;
            __stcg(a.part_ml + at, mine ? make_float2(m, l) : make_float2(-INFINITY, 0.0f));
        }
#pragma unroll 1
        for (uint32_t c = 0; c < HD / 32; ++c) {
            float o[32];
            if (mine && ok) {
                tmem_ld32(to + c * 32, o);
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = 0.0f;
            }
            if (valid) {
                float4* d = reinterpret_cast<float4*>(a.part_o + at * HD + c * 32);
#pragma unroll
                for (int i = 0; i < 8; ++i) __stcg(d + i, make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]));
            }
        }
    } else if (warp < 12) {
        // ---- copies: slots take K0 V0 K1 V1 ...; a warp brings 32 rows of each -----------------
        const uint32_t lw = warp - 8;
        constexpr uint32_t RP = 32 / CH;       // rows of one instruction
        constexpr uint32_t N = 32 / RP;        // instructions for the warp's 32 rows
        constexpr uint32_t AHEAD = NS - 2;     // slots under way before the oldest is waited for
        const uint32_t lr = lane / CH, lc = lane % CH;
        const T* bases[2] = {reinterpret_cast<const T*>(a.k), reinterpret_cast<const T*>(a.v)};
        bool alive = true;
        uint32_t fill = 0, done = 0;
        auto finish = [&] {  // the oldest slot's copies are visible to the tensor core
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[done % NS]);
            ++done;
        };
        for (uint32_t tile = 0; tile < n_tiles && alive; ++tile) {
            const uint32_t row = w.r0 + tile * TC_ROWS + lw * 32 + lane;
            uint64_t off;
            if (!(row < w.r1 && attn_row(a, w, head, row, off))) off = ~0ull;  // zeros
#pragma unroll
            for (int kv = 0; kv < 2; ++kv, ++fill) {
                const uint32_t slot = fill % NS;
                if (fill >= NS) {
                    alive = __all_sync(0xffffffffu, mbar_wait(&empty[slot], (fill / NS - 1) & 1, QDEV_WAIT_EMPTY_TIMEOUT));
                    if (!alive) break;
                }
                const uint32_t st = s_kv + slot * S::TILE;
#pragma unroll
                for (uint32_t p = 0; p < N; ++p) {
                    const uint32_t rw = p * RP + lr, r = lw * 32 + rw;
                    const uint64_t o = __shfl_sync(0xffffffffu, off, rw);
                    const uint32_t at = st + (lc >> 3) * S::PANEL + r * 128 + (((lc & 7) ^ (r & 7)) << 4);
                    cp_async16(at, bases[kv] + (o == ~0ull ? 0ull : o) + lc * 8, o == ~0ull ? 0u : 16u);
                }
                cp_async_commit();
                if (fill - done >= AHEAD) {
                    cp_async_wait<AHEAD>();
                    finish();
                }
            }
        }
        cp_async_wait_all();
        while (done < fill && alive) finish();
    } else if (lane == 0) {
        // ---- products ---------------------------------------------------------------------------
        bool alive = true;
        auto wait = [&](uint64_t* bar, uint32_t parity) {
            if (alive) alive = mbar_wait(bar, parity, QDEV_WAIT_FULL_TIMEOUT);
            tc_fence_after();
        };
        auto qk = [&](uint32_t t, uint32_t tile) {
            const uint32_t q = s_q + (pair ? t * S::TILE : 0), k = s_kv + ((2 * tile) % NS) * S::TILE;
#pragma unroll
            for (uint32_t j = 0; j < HD / 16; ++j) {
                const uint32_t at = (j >> 2) * S::PANEL + (j & 3) * 32;
                umma_f16(tmem + t * 128, umma_desc_sw128(q + at), umma_desc_sw128(k + at), j != 0, ID_QK);
            }
            umma_commit(&s_full[t]);
        };
        auto pv = [&](uint32_t t, uint32_t tile, bool first) {
            const uint32_t v = s_kv + ((2 * tile + 1) % NS) * S::TILE;
#pragma unroll
            for (uint32_t j = 0; j < TC_ROWS / 16; ++j)
                umma_f16_ta(tmem + 256 + t * 128, tmem + t * 128 + j * 8, umma_desc_sw128_mn(v + j * 2048, S::PANEL), !(first && j == 0), ID_PV);
        };
        auto k_full = [&](uint32_t tile) { wait(&full[(2 * tile) % NS], (2 * tile / NS) & 1); };
        auto v_full = [&](uint32_t tile) { wait(&full[(2 * tile + 1) % NS], ((2 * tile + 1) / NS) & 1); };
        auto k_free = [&](uint32_t tile) { umma_commit(&empty[(2 * tile) % NS]); };
        auto v_free = [&](uint32_t tile) { umma_commit(&empty[(2 * tile + 1) % NS]); };
        if (n_tiles) wait(q_full, 0);
        if (pair) {
            if (n_tiles) {
                k_full(0);
                if (alive) {
                    qk(0, 0);
                    qk(1, 0);
                    k_free(0);
                }
            }
            for (uint32_t i = 0; i < n_tiles && alive; ++i) {
                const bool more = i + 1 < n_tiles;
                v_full(i);
                if (more) k_full(i + 1);
                for (uint32_t t = 0; t < 2; ++t) {
                    wait(&p_full[t], i & 1);
                    if (!alive) break;
                    pv(t, i, i == 0);
                    if (t) v_free(i);
                    if (more) qk(t, i + 1);
                    else umma_commit(&o_full[t]);
                    if (more && t) k_free(i + 1);
                }
            }
        } else {
            for (uint32_t t = 0; t < 2 && t < n_tiles; ++t) {
                k_full(t);
                if (!alive) break;
                qk(t, t);
                k_free(t);
            }
            for (uint32_t i = 0; i < n_tiles && alive; ++i) {
                const uint32_t t = i & 1;
                v_full(i);
                wait(&p_full[t], (i >> 1) & 1);
                if (!alive) break;
                pv(t, i, i < 2);
                v_free(i);
                if (i + 2 < n_tiles) {
                    k_full(i + 2);
                    if (!alive) break;
                    qk(t, i + 2);
                    k_free(i + 2);
                } else {
                    umma_commit(&o_full[t]);
                }
            }
        }
        // every product issued has finished before TMEM is freed
        if (n_tiles) {
            umma_commit(drain);
            mbar_wait(drain, 0, QDEV_WAIT_FULL_TIMEOUT);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 12) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

}  // namespace qb200
