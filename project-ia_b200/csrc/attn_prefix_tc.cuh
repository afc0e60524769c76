// attn_prefix_tc.cuh — the shared prefix's pass on tcgen05 (fp16 and bf16
// caches, head_dim 64 or 128).
//
// All new tokens' query vectors of a KV head (tokens x G heads) meet the same
// rows, so the pass is a matrix product: S = Q K^T and O += P V with 128
// query vectors as the MMA's M, 128 rows of the cache as one tile.  One CTA
// runs two streams, each with scores and an output of its own in TMEM:
//   two tiles of vectors, the same rows (more than 128 vectors), or
//   one tile of vectors, even and odd row tiles (up to 128; joined at the end),
// so that one stream's products run while the other's exponentials do
// (columns: S at 128 stream, O at 256 + 128 stream).  A stream's exponentials
// come in two halves of 64 rows, so that the first half's product with V runs
// beside the second half's exponentials.
//
// Roles: warps 0-3 and 4-7 are the streams' softmax, a thread per vector
// (its row of S lies in its own TMEM lane, so maximum and sum need no
// exchange); warps 8-11 copy rows of K and V (16-byte cp.async into the
// 128-byte swizzle that the MMA's descriptors name; a row's page is looked up
// by one lane); warp 13 hands landed tiles over to the tensor core's proxy;
// warp 12 issues the products.  P overwrites S
// in TMEM in 16 bits (the operand type) and is the A operand of P V from
// there; V is used as it lies in the cache, [row][dim], as an MN-major B
// operand.
//
// Tried: scores of 64 rows with two buffers a stream, instead of 128 with one,
// keep a stream's exponentials apart from its own products, but a product of
// 64 columns takes 57 clocks where one of 128 takes 64 (operands come from
// shared memory at 128 bytes a clock).  A warp that polls both streams and
// takes whichever is ready spends 3000 clocks a tile on doing so.
//
// The reference of the weights (attn_reference) moves seldom: then the output
// is rescaled in TMEM.
//
// Bound: for up to 128 vectors the bytes of K and V; beyond, the tensor pipe
// (4 x 128 x 128 x head_dim flops a tile and stream) with the exponentials (128
// x 128 of them, a quarter on the multiply-add units) in its way: 512 vectors x
// 32768 rows x 8 KV heads of 128 take 78 us by themselves, 0.88 PFLOP/s with the
// tensor pipe busy half of the time: 29 tiles a CTA at 3450 clocks, of which the
// pipe works 2048 (62 us at the 1.66 GHz that the power cap leaves), and a CTA's
// begin and end.
#pragma once

#include "attn_prefix.cuh"
#include "prefill.cuh"

namespace qb200 {

static constexpr uint32_t TC_THREADS = 448;
static constexpr uint32_t TC_ROWS = 128, TC_HALF = 64;

template <int HD>
struct TcShape {
    static constexpr uint32_t SLOTS = HD == 128 ? 5 : 9;        // K and V tiles in the ring
    static constexpr uint32_t TILE = TC_ROWS * HD * 2;          // one K or V tile, one tile of Q
    static constexpr uint32_t PANEL = TC_ROWS * 128;            // 64 columns of it
    static constexpr size_t SMEM = (size_t)(2 + SLOTS) * TILE + 1024 + 512;
    static_assert(SLOTS * TILE >= 256 * (HD + 4) * 4 + 1024, "the outputs fit into the ring");
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

// True in one lane of the warp, always the same one.
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}

// 2^x for two numbers on the multiply-add units: x = k + f with |f| <= 1/2 (x
// + 1.5 * 2^23 rounds there), the exponential's series to f^4 (off by 5.6e-5
// of the value, a ninth of fp16's half step), and k added to the exponent.
// 2^-127 and all below it come out as zero, as a score of -infinity has to;
// between there and 2^-126 it is something up to 2^-126.
__device__ __forceinline__ F2 ex2_series(F2 x) {
    float a, b, p, q, s, t;
    x.get(a, b);
    x = F2(fmaxf(a, -127.0f), fmaxf(b, -127.0f));
    const F2 big(12582912.0f, 12582912.0f), r = add2(x, big);
    const F2 f = sub2(x, sub2(r, big));
    F2 e = fma2(f, F2(0.00961813f, 0.00961813f), F2(0.05550411f, 0.05550411f));
    e = fma2(e, f, F2(0.24022651f, 0.24022651f));
    e = fma2(e, f, F2(0.69314718f, 0.69314718f));
    e = fma2(e, f, F2(1.0f, 1.0f));
    e.get(p, q);
    r.get(s, t);
    return F2(__uint_as_float(__float_as_uint(p) + (__float_as_uint(s) << 23)), __uint_as_float(__float_as_uint(q) + (__float_as_uint(t) << 23)));
}

// The largest of three, NaN if one of them is.
__device__ __forceinline__ float max_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// 16 and 64 consecutive columns of this warp's 32 TMEM lanes.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
#define TC_R16(b) \
    "=r"(r[b]), "=r"(r[b + 1]), "=r"(r[b + 2]), "=r"(r[b + 3]), "=r"(r[b + 4]), "=r"(r[b + 5]), "=r"(r[b + 6]), "=r"(r[b + 7]), \
        "=r"(r[b + 8]), "=r"(r[b + 9]), "=r"(r[b + 10]), "=r"(r[b + 11]), "=r"(r[b + 12]), "=r"(r[b + 13]), "=r"(r[b + 14]), "=r"(r[b + 15])
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, uint32_t (&r)[64]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
        "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,"
        "%62,%63}, [%64];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : TC_R16(0), TC_R16(16), TC_R16(32), TC_R16(48)
        : "r"(taddr)
        : "memory");
}
#undef TC_R16

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
    uint64_t* landed = full + NS;
    uint64_t* empty = landed + NS;
    uint64_t* s_full = empty + NS;  // [stream]: scores are there
    uint64_t* p_full = s_full + 2;  // [stream][half]: exponentials are
    uint64_t* o_done = p_full + 4;  // [stream]: a half's product with V is done
    uint64_t* o_last = o_done + 2;  // [stream]: the last one is
    uint64_t* q_full = o_last + 2;
    uint64_t* drain = q_full + 1;   // every product is done
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);

    const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, head = blockIdx.z, split = blockIdx.x;
    const bool pair = !a.alternate;  // two tiles of vectors

    if (tid == 0) {
        for (uint32_t i = 0; i < NS; ++i) {
            mbar_init(&landed[i], 128);  // each copying thread's copies
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int t = 0; t < 4; ++t) mbar_init(&p_full[t], 4);
        mbar_init(&s_full[0], 1);
        mbar_init(&s_full[1], 1);
        for (int t = 0; t < 2; ++t) {
            mbar_init(&o_done[t], 1);
            mbar_init(&o_last[t], 1);
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
    // barriers and TMEM are set up beside the tail of the stream's work before this pass
    pdl_wait();
    pdl_trigger();  // the pass over the own rows may start beside this one
    AttnItem w;
    const bool any = attn_item(a, blockIdx.y, split, pair ? 256 : 128, TC_ROWS, w);
    const uint32_t n_tiles = any ? (w.r1 - w.r0 + TC_ROWS - 1) / TC_ROWS : 0;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp < 8) {
        // ---- softmax ----------------------------------------------------------------------
        const uint32_t t = warp >> 2, row = tid & 127;
        const uint32_t lanes = tmem + (((warp & 3) * 32u) << 16), to = lanes + 256 + t * 128;
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
        const F2 c2(a.c, a.c);
        float m = -INFINITY;
        F2 sum;  // of even and odd columns
        bool alive = true;
        for (uint32_t u = 0; u < 2 * mine && alive; ++u) {  // half tiles
            const uint32_t j = u >> 1, h = u & 1, ts = lanes + t * 128 + h * TC_HALF;
            if (h == 0) {
                alive = __all_sync(0xffffffffu, mbar_wait(&s_full[t], j & 1, QDEV_WAIT_FULL_TIMEOUT));
                if (!alive) break;
                tc_fence_after();
            }
            uint32_t v[64];
            tmem_ld64(ts, v);
            const int32_t cols = (int32_t)(w.r1 - w.r0) - (int32_t)((pair ? j : 2 * j + t) * TC_ROWS + h * TC_HALF);
            if (cols < (int32_t)TC_HALF) {  // rows past the end score nothing
#pragma unroll
                for (int i = 0; i < 64; ++i)
                    if (i >= cols) v[i] = 0xff800000u;
            }
            float mx = -INFINITY, my = -INFINITY;
#pragma unroll
            for (int i = 0; i < 64; i += 4) {
                mx = max_nan(mx, __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
                my = max_nan(my, __uint_as_float(v[i + 2]), __uint_as_float(v[i + 3]));
            }
            mx = max_nan(mx, my, my) * a.c;  // c > 0
            // a score that is no number or infinite: so is the sum, and every output (the series' clamp would hide a NaN)
            const bool lost = !(mx < INFINITY);
            const float M = attn_reference<T>(m, mx);  // NaN moves nothing
            const bool move = M != m;                  // also from -infinity
            if (__any_sync(0xffffffffu, move)) {
                const float f = move ? (m == -INFINITY ? 0.0f : ex2(m - M)) : 1.0f;
                m = M;
                float s0, s1;
                sum.get(s0, s1);
                sum = F2(s0 * f, s1 * f);
                if (u > 0) {  // the product before this one is done before its output is touched
                    alive = __all_sync(0xffffffffu, mbar_wait(&o_done[t], (u - 1) & 1, QDEV_WAIT_FULL_TIMEOUT));
                    if (!alive) break;
                    tc_fence_after();
#pragma unroll 1
                    for (uint32_t c = 0; c < HD / 16; ++c) {
                        uint32_t o[16];
                        tmem_ld16(to + c * 16, o);
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                        tmem_st16(to + c * 16, o);
                    }
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                }
            }
            const float sub = m == -INFINITY ? 0.0f : -m;
            const F2 sub2f(sub, sub);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                uint32_t p[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float x, y;
                    F2 e = fma2(F2(__uint_as_float(v[32 * k + 2 * i]), __uint_as_float(v[32 * k + 2 * i + 1])), c2, sub2f);
                    if (i % 4 == 3) {  // a quarter beside the special function unit
                        e = ex2_series(e);
                        e.get(x, y);
                    } else {
                        e.get(x, y);
                        x = ex2(x);
                        y = ex2(y);
                        e = F2(x, y);
                    }
                    sum = add2(sum, e);
                    p[i] = pack2<T>(x, y);
                }
                tmem_st16(ts + k * 16, p);
            }
            if (lost) sum = F2(__int_as_float(0x7fffffff), 0.0f);
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[2 * t + h]);
        }
        float l, l1;
        sum.get(l, l1);
        l += l1;
        // ---- this stream's part ----
        bool ok = alive && mine;
        // (a barrier of its own: o_done may be one phase back or two by now, which a parity cannot tell)
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&o_last[t], 0, QDEV_WAIT_FULL_TIMEOUT));
        tc_fence_after();
        if (!ok) m = -INFINITY, l = 0.0f;
        const uint32_t v = (pair ? t * 128 : 0) + row;
        const bool valid = any && v < w.n_vec;
        // Both streams' products are done behind this barrier, so the ring's place takes the outputs, a
        // row of HD + 4 floats per vector (16-byte accesses of neighbouring rows meet different banks),
        // which one bulk copy each takes to the workspace (rows of 16-byte stores from TMEM took 5 us).
        asm volatile("bar.sync 2, 256;" ::: "memory");
        constexpr uint32_t OP = HD + 4;
        float* s_o = reinterpret_cast<float*>(smem + 2 * S::TILE);  // [2][128][OP]
        float* mine_o = s_o + (t * 128 + row) * OP;
        float* s_ml = s_o + 256 * OP;                               // [128][2]
        auto stage = [&](float f0, const float* other, float f1) {
#pragma unroll 1
            for (uint32_t c = 0; c < HD / 16; ++c) {
                uint32_t o[16];
                if (ok) tmem_ld16(to + c * 16, o);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (ok) x = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]), __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
                    if (other) {
                        const float4 y = *reinterpret_cast<const float4*>(other + c * 16 + 4 * i);
                        x = make_float4(x.x * f0 + y.x * f1, x.y * f0 + y.y * f1, x.z * f0 + y.z * f1, x.w * f0 + y.w * f1);
                    }
                    *reinterpret_cast<float4*>(mine_o + c * 16 + 4 * i) = x;
                }
            }
        };
        if (pair || t == 1) stage(1.0f, nullptr, 0.0f);
        if (!pair) {  // the second stream's share goes through shared memory to the first
            if (t == 1) {
                s_ml[row * 2] = m;
                s_ml[row * 2 + 1] = l;
            }
            asm volatile("bar.sync 2, 256;" ::: "memory");
            if (t == 0) {
                const float m1 = s_ml[row * 2], l2 = s_ml[row * 2 + 1], M = fmaxf(m, m1);
                const float f0 = m == M ? 1.0f : ex2(m - M), f1 = m1 == M ? 1.0f : ex2(m1 - M);
                m = M;
                l = l * f0 + l2 * f1;
                stage(f0, s_o + (128 + row) * OP, f1);
            }
        }
        if (valid && (pair || t == 0)) {
            const uint32_t i = fast_div(w.vec0 + v, a.by_group), h = head * a.group + (w.vec0 + v - i * a.group);
            const uint64_t at = ((uint64_t)split * a.n_tokens + i) * a.n_heads + h;
            __stcg(a.part_ml + at, make_float2(m, l));
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(a.part_o + at * HD), "r"(smem_u32(mine_o)), "r"(HD * 4) : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        }
    } else if (warp < 12) {
        // ---- copies: slots take K0 V0 K1 V1 ...; a warp brings 32 rows of each -----------------
        const uint32_t lw = warp - 8;
        constexpr uint32_t RP = 32 / CH;       // rows of one instruction
        constexpr uint32_t N = 32 / RP;        // instructions for the warp's 32 rows
        const uint32_t lr = lane / CH, lc = lane % CH;
        const T* bases[2] = {reinterpret_cast<const T*>(a.k), reinterpret_cast<const T*>(a.v)};
        bool alive = true;
        uint32_t fill = 0;
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
                cp_async_arrive(&landed[slot]);
            }
        }
        cp_async_wait_all();
    } else if (warp == 13) {
        // ---- landed copies, generic-proxy writes of other threads, to the tensor core's proxy ----------
        bool alive = true;
        for (uint32_t f = 0; f < 2 * n_tiles && alive; ++f) {
            alive = __all_sync(0xffffffffu, mbar_wait(&landed[f % NS], (f / NS) & 1, QDEV_WAIT_FULL_TIMEOUT));
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            if (alive && lane == 0) mbar_arrive(&full[f % NS]);
        }
    } else {
        // ---- products ---------------------------------------------------------------------------
        // The whole warp takes these steps and one elected lane issues: what a product needs (addresses,
        // descriptors) is then the same in all lanes and stays in uniform registers, where the
        // instruction reads it.  Formed by a single lane in a branch of its own, the 48 products of a
        // tile took 5100 clocks to issue.
        // Every instruction here is on the streams' way (a state machine that polled both streams took
        // 3000 clocks a tile), so slots are counted, not divided.
        bool alive = true;
        const uint32_t tiles = __shfl_sync(0xffffffffu, n_tiles, 0), tm = __shfl_sync(0xffffffffu, tmem, 0);
        const uint64_t hi = umma_desc_sw128(0) & ~0xffffffffull;  // of every descriptor here
        const uint32_t lo_k = (uint32_t)umma_desc_sw128(0), lo_mn = (uint32_t)umma_desc_sw128_mn(0, S::PANEL);
        struct Slot {  // of the K or V tile that is used next
            uint32_t at, phase;
            __device__ __forceinline__ void next(uint32_t by) {
                at += by;
                if (at >= NS) {
                    at -= NS;
                    phase ^= 1;
                }
            }
        };
        auto wait = [&](uint64_t* bar, uint32_t parity) {
            if (alive) alive = __all_sync(0xffffffffu, mbar_wait(bar, parity, QDEV_WAIT_FULL_TIMEOUT));
            tc_fence_after();
        };
        auto qk = [&](uint32_t t, uint32_t slot, uint64_t* free_k) {
            const uint32_t lq = lo_k + ((s_q + (pair ? t * S::TILE : 0)) >> 4), lk = lo_k + ((s_kv + slot * S::TILE) >> 4);
            const uint32_t d = tm + t * 128;
            if (elect_one()) {
#pragma unroll
                for (uint32_t j = 0; j < HD / 16; ++j) {
                    const uint32_t at = ((j >> 2) * S::PANEL + (j & 3) * 32) >> 4;  // added to the address field
                    umma_f16(d, hi | (lq + at), hi | (lk + at), j != 0, ID_QK);
                }
                umma_commit(&s_full[t]);
                if (free_k) umma_commit(free_k);
            }
            __syncwarp();
        };
        auto pv = [&](uint32_t t, uint32_t slot, uint32_t h, bool first, bool last, uint64_t* free_v) {
            const uint32_t lv = lo_mn + ((s_kv + slot * S::TILE + h * TC_HALF * 128) >> 4);
            const uint32_t d = tm + 256 + t * 128, p = tm + t * 128 + h * TC_HALF;
            if (elect_one()) {
#pragma unroll
                for (uint32_t j = 0; j < TC_HALF / 16; ++j) umma_f16_ta(d, p + j * 8, hi | (lv + j * (2048 >> 4)), !(first && j == 0), ID_PV);
                umma_commit(last ? &o_last[t] : &o_done[t]);
                if (free_v) umma_commit(free_v);
            }
            __syncwarp();
        };
        Slot k = {0, 0}, v = {1, 0};
        if (tiles) wait(q_full, 0);
        if (pair) {
            if (tiles) {
                wait(&full[k.at], k.phase);
                if (alive) {
                    qk(0, k.at, nullptr);
                    qk(1, k.at, &empty[k.at]);
                }
            }
            for (uint32_t i = 0; i < tiles && alive; ++i) {
                const bool more = i + 1 < tiles;
                k.next(2);
                wait(&full[v.at], v.phase);
                wait(&p_full[0], i & 1);
                if (!alive) break;
                pv(0, v.at, 0, i == 0, false, nullptr);
                wait(&p_full[2], i & 1);
                if (!alive) break;
                pv(1, v.at, 0, i == 0, false, nullptr);
                if (more) wait(&full[k.at], k.phase);
                wait(&p_full[1], i & 1);
                if (!alive) break;
                pv(0, v.at, 1, false, !more, nullptr);
                if (more) qk(0, k.at, nullptr);
                wait(&p_full[3], i & 1);
                if (!alive) break;
                pv(1, v.at, 1, false, !more, &empty[v.at]);
                if (more) qk(1, k.at, &empty[k.at]);
                v.next(2);
            }
        } else {
            for (uint32_t t = 0; t < 2 && t < tiles && alive; ++t) {
                wait(&full[k.at], k.phase);
                if (alive) qk(t, k.at, &empty[k.at]);
                k.next(2);
            }
            for (uint32_t i = 0; i < tiles && alive; ++i) {
                const uint32_t t = i & 1, par = (i >> 1) & 1;
                wait(&full[v.at], v.phase);
                wait(&p_full[2 * t], par);
                if (!alive) break;
                pv(t, v.at, 0, i < 2, false, nullptr);
                wait(&p_full[2 * t + 1], par);
                if (!alive) break;
                pv(t, v.at, 1, false, i + 2 >= tiles, &empty[v.at]);
                v.next(2);
                if (i + 2 < tiles) {
                    wait(&full[k.at], k.phase);
                    if (!alive) break;
                    qk(t, k.at, &empty[k.at]);
                    k.next(2);
                }
            }
        }
        // every product issued has finished before TMEM is freed
        if (tiles) {
            if (elect_one()) umma_commit(drain);
            __syncwarp();
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
