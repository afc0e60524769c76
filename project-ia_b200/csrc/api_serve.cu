// api_serve.cu — the serving operators' entry points: argument checks, plans
// and launches (kernels: rotate.cuh, attn_prefix.cuh, verify.cuh).
//
// Every launch is a programmatic dependent one: a kernel's CTAs may be set up
// beside the tail of the work before it, and wait for that work's end before
// they read or write.  Nothing is allocated and nothing is kept between calls; checks that need
// no device come first, so that a refusal is the same with and without one.
#include <cmath>

#include "attn_few.cuh"
#include "attn_prefix.cuh"
#include "attn_prefix_tc.cuh"
#include "runtime.cuh"
#include "verify.cuh"

using namespace qb200;

namespace {

constexpr uint32_t SMS = 148;  // of a B200; plans are made without a device too

uint32_t size_of(uint32_t dtype) { return dtype == Q_B200_F32 ? 4u : 2u; }
bool known(uint32_t dtype) { return dtype <= Q_B200_BF16; }

// Device memory (or managed memory) of the current device: a host pointer or
// another GPU's would fault in the kernel.
struct DevicePtrs {
    int dev = -1;
    bool ok = true;
    DevicePtrs() { ok = cuda_ok(cudaGetDevice(&dev), "cudaGetDevice"); }
    DevicePtrs& operator()(const void* p) {
        if (!ok || !p) return *this;
        cudaPointerAttributes at;
        ok = cuda_ok(cudaPointerGetAttributes(&at, p), "cudaPointerGetAttributes");
        if (ok && !(at.type == cudaMemoryTypeManaged || (at.type == cudaMemoryTypeDevice && at.device == dev))) {
            set_last_error("a pointer is not of the current device", cudaErrorInvalidValue);
            ok = false;
        }
        return *this;
    }
};

FastDiv fast_div_of(uint32_t d) {
    uint32_t s = 0;
    while ((1ull << s) < d) ++s;
    return {d, (uint32_t)(((1ull << 32) * ((1ull << s) - d)) / d + 1), s};
}

uint32_t cdiv(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1) / b); }

uint64_t align_of(std::initializer_list<uint64_t> v) {  // largest power of two that divides all
    uint64_t all = 0;
    for (uint64_t x : v) all |= x;
    return all ? (all & (~all + 1)) : ~0ull;
}
// Strides that kernels keep in 32 bits.
bool short_strides(std::initializer_list<uint64_t> v) {
    for (uint64_t x : v)
        if (x >> 32) return false;
    return true;
}
uint64_t addr(const void* p) { return (uint64_t)(uintptr_t)p; }

bool overlap(const void* a, uint64_t an, const void* b, uint64_t bn) {
    return a && b && an && bn && addr(a) < addr(b) + bn && addr(b) < addr(a) + an;
}

q_error_code check_cache(const q_b200_paged_kv& kv) {
    if (!kv.k || !kv.v) return Q_ERR_INVALID_ARG;
    if (!known(kv.dtype)) return Q_ERR_INVALID_DTYPE;
    if (kv.reserved) return Q_ERR_INVALID_ARG;
    if (kv.n_pages == 0 || kv.page_rows == 0 || kv.n_kv_heads == 0 || kv.head_dim == 0) return Q_ERR_INVALID_SIZE;
    if (kv.page_rows > (1u << 30) || !short_strides({kv.head_stride, kv.row_stride})) return Q_ERR_INVALID_SIZE;
    if (kv.row_stride < kv.head_dim && kv.page_rows > 1) return Q_ERR_INVALID_SIZE;
    if ((addr(kv.k) | addr(kv.v)) & (size_of(kv.dtype) - 1)) return Q_ERR_MISALIGNED;
    return Q_OK;
}

q_error_code check_plan(const q_b200_rope_plan* p, uint32_t head_dim) {
    if (p->rot_dim < 2 || p->rot_dim > 256 || p->rot_dim % 2 || p->rot_dim > head_dim) return Q_ERR_INVALID_SIZE;
    if (p->layout > Q_B200_ROPE_HALF) return Q_ERR_INVALID_ARG;
    return Q_OK;
}

// ---- rotation -------------------------------------------------------------------

template <typename TI, typename TC, int E>
cudaError_t launch_rotate_units(RotateArgs& a, cudaStream_t st) {
    a.rot_units = a.rot / (2 * E);
    const uint32_t U = a.rot_units + (a.head_dim - a.rot) / E;
    a.heads = a.part[0].heads + a.part[1].heads + a.part[2].heads;
    // Two or three units a thread, whichever whole tokens fill better, where
    // that fills the GPU; else one, for the shortest path through few tokens.
    a.row_step = ROT_THREADS / U;  // U <= 256: head_dim is
    const uint64_t all = (uint64_t)a.n_tokens * a.heads * U;
    const uint32_t most = a.rot ? std::min(ROT_TOKENS, ROT_ANGLES / (a.rot / 2)) : ROT_TOKENS;
    uint32_t N = 0, filled = 0;
    for (uint32_t n = all >= 8ull * SMS * ROT_THREADS ? 2 : 1, last = n == 1 ? 1 : 3; n <= last; ++n) {
        const uint32_t room = n * a.row_step, h = std::min(a.heads, room), t = std::min({a.n_tokens, std::max(1u, room / h), most});
        if (N && h * t * 1000 / room <= filled) continue;
        N = n;
        filled = h * t * 1000 / room;
        a.cta_heads = h;
        a.cta_tokens = t;
    }
    a.by_units = fast_div_of(U);
    a.by_heads = fast_div_of(a.cta_heads);
    a.by_pairs = fast_div_of(std::max(1u, a.rot / 2));
    const dim3 grid(cdiv(a.n_tokens, a.cta_tokens), cdiv(a.heads, a.cta_heads));
    auto go = [&](auto append) {
        constexpr bool A = decltype(append)::value;
        return launch_ex(N == 3 ? rotate_kernel<TI, TC, E, 3, A> : N == 2 ? rotate_kernel<TI, TC, E, 2, A> : rotate_kernel<TI, TC, E, 1, A>,
                         grid, dim3(ROT_THREADS), 0, st, true, a);
    };
    if constexpr (std::is_same<TI, TC>::value)
        if (!a.row) return go(std::false_type());
    return go(std::true_type());  // q_b200_kv_append; types that differ are its alone
}

template <typename TI, typename TC>
cudaError_t launch_rotate(RotateArgs& a, uint32_t E, cudaStream_t st) {
    if constexpr (sizeof(TI) == 2 || sizeof(TC) == 2)
        if (E == 8) return launch_rotate_units<TI, TC, 8>(a, st);
    return E == 4 ? launch_rotate_units<TI, TC, 4>(a, st) : launch_rotate_units<TI, TC, 1>(a, st);
}

RotateRows rotate_rows(const void* src, void* dst, uint64_t st, uint64_t sh, uint64_t dt, uint64_t dh, uint32_t heads,
                       bool rotate) {
    return {src, dst, (uint32_t)st, (uint32_t)sh, (uint32_t)dt, (uint32_t)dh, heads, rotate ? 1u : 0u};
}

void set_plan(RotateArgs& a, const q_b200_rope_plan* plan, bool transpose) {
    a.rot = plan ? plan->rot_dim : 0;
    a.interleaved = plan && plan->layout == Q_B200_ROPE_INTERLEAVED;
    a.gain = plan ? plan->gain : 1.0f;
    a.sign = transpose ? -a.gain : a.gain;
    if (plan) std::memcpy(a.turns, plan->turns, sizeof(double) * (plan->rot_dim / 2));
}

// Elements of a vector: as many as 16 bytes of the narrowest type hold, if
// every row part begins on such a vector (`by`: the divisor in bytes of all
// addresses and strides of elements of `es` bytes) and the row divides.
bool vectors_fit(uint32_t E, uint32_t es, uint64_t by, const RotateArgs& a) {
    if (by < std::min<uint64_t>(16, (uint64_t)E * es)) return false;
    const uint32_t pair = a.interleaved ? a.rot % (2 * E) : (a.rot / 2) % E;
    return pair == 0 && (a.head_dim - a.rot) % E == 0;
}

}  // namespace

extern "C" {

q_error_code q_b200_rope_plan_init(q_b200_rope_plan* plan, uint32_t rot_dim, q_b200_rope_layout layout, double base,
                                   const q_b200_rope_scale* scale) {
    if (!plan) return Q_ERR_INVALID_ARG;
    if (rot_dim < 2 || rot_dim > 256 || rot_dim % 2) return Q_ERR_INVALID_SIZE;
    if ((uint32_t)layout > Q_B200_ROPE_HALF || !(base > 1.0) || !std::isfinite(base)) return Q_ERR_INVALID_ARG;
    const uint32_t kind = scale ? scale->kind : (uint32_t)Q_B200_ROPE_PLAIN;
    if (kind > Q_B200_ROPE_YARN || (scale && scale->reserved)) return Q_ERR_INVALID_ARG;
    if (kind != Q_B200_ROPE_PLAIN && !(scale->factor > 0.0 && std::isfinite(scale->factor))) return Q_ERR_INVALID_ARG;
    if (kind >= Q_B200_ROPE_BANDED &&
        !(scale->original_len > 0.0 && scale->low > 0.0 && scale->high > scale->low && std::isfinite(scale->high) &&
          std::isfinite(scale->original_len)))
        return Q_ERR_INVALID_ARG;
    if (kind == Q_B200_ROPE_YARN && !(scale->gain >= 0.0 && std::isfinite(scale->gain))) return Q_ERR_INVALID_ARG;
    const double tau = 6.283185307179586476925286766559;
    std::memset(plan, 0, sizeof *plan);
    plan->rot_dim = rot_dim;
    plan->layout = layout;
    plan->gain = 1.0f;
    double low = 0.0, high = 0.0;
    if (kind == Q_B200_ROPE_YARN) {
        // pair index whose wave turns n times in original_len
        auto pair_of = [&](double n) { return rot_dim * std::log(scale->original_len / (n * tau)) / (2.0 * std::log(base)); };
        low = std::max(std::floor(pair_of(scale->high)), 0.0);
        high = std::min(std::ceil(pair_of(scale->low)), (double)rot_dim - 1.0);
        plan->gain = (float)(scale->gain > 0.0 ? scale->gain : 0.1 * std::log(scale->factor) + 1.0);
    }
    for (uint32_t i = 0; i < rot_dim / 2; ++i) {
        double f = std::pow(base, -2.0 * i / rot_dim);
        if (kind == Q_B200_ROPE_LINEAR) {
            f /= scale->factor;
        } else if (kind == Q_B200_ROPE_BANDED) {
            const double turns = scale->original_len * f / tau;
            const double s = std::min(std::max((turns - scale->low) / (scale->high - scale->low), 0.0), 1.0);
            f = (1.0 - s) * f / scale->factor + s * f;
        } else if (kind == Q_B200_ROPE_YARN) {
            const double s = std::min(std::max((i - low) / std::max(high - low, 0.001), 0.0), 1.0);
            f = f / scale->factor * s + f * (1.0 - s);
        }
        plan->turns[i] = f / tau;
    }
    return Q_OK;
}

q_error_code q_b200_rope(const q_b200_rope_args* r, void* stream) {
    if (!r || !r->x || !r->out || !r->pos || !r->plan) return Q_ERR_INVALID_ARG;
    if (!known(r->dtype)) return Q_ERR_INVALID_DTYPE;
    if (r->reserved || r->transpose > 1) return Q_ERR_INVALID_ARG;
    if (r->n_tokens == 0 || r->n_heads == 0 || r->n_heads > 65535 || r->head_dim == 0 || r->head_dim > 256)
        return Q_ERR_INVALID_SIZE;
    if (q_error_code rc = check_plan(r->plan, r->head_dim)) return rc;
    const uint32_t es = size_of(r->dtype);
    if (((addr(r->x) | addr(r->out)) & (es - 1)) || (addr(r->pos) & 3)) return Q_ERR_MISALIGNED;
    if (!short_strides({r->x_token_stride, r->x_head_stride, r->out_token_stride, r->out_head_stride})) return Q_ERR_INVALID_SIZE;
    // in place means the same elements; another overlay would be read after it is written
    if (r->x == r->out && (r->x_token_stride != r->out_token_stride || r->x_head_stride != r->out_head_stride))
        return Q_ERR_ALIASING;
    if (!DevicePtrs()(r->x)(r->out)(r->pos).ok) return Q_ERR_INVALID_ARG;
    RotateArgs a{};
    set_plan(a, r->plan, r->transpose != 0);
    a.pos = r->pos;
    a.n_tokens = r->n_tokens;
    a.head_dim = r->head_dim;
    a.part[2] = rotate_rows(r->x, r->out, r->x_token_stride, r->x_head_stride, r->out_token_stride, r->out_head_stride,
                            r->n_heads, true);
    const uint64_t by = align_of({addr(r->x), addr(r->out), r->x_token_stride * es, r->x_head_stride * es,
                                  r->out_token_stride * es, r->out_head_stride * es});
    uint32_t E = es == 4 ? 4 : 8;
    while (E > 1 && !vectors_fit(E, es, by, a)) E = E == 8 ? 4 : 1;
    cudaStream_t st = (cudaStream_t)stream;
    switch (r->dtype) {
        case Q_B200_F32: Q_CUDA((launch_rotate<float, float>(a, E, st))); break;
        case Q_B200_F16: Q_CUDA((launch_rotate<__half, __half>(a, E, st))); break;
        default: Q_CUDA((launch_rotate<__nv_bfloat16, __nv_bfloat16>(a, E, st))); break;
    }
    return Q_OK;
}

q_error_code q_b200_kv_append(const q_b200_append_args* r, void* stream) {
    if (!r || !r->k || !r->v || !r->pages || !r->row) return Q_ERR_INVALID_ARG;
    if (q_error_code rc = check_cache(r->kv)) return rc;
    if (!known(r->dtype)) return Q_ERR_INVALID_DTYPE;
    if (r->reserved || (r->q && !r->q_out)) return Q_ERR_INVALID_ARG;
    if (r->n_tokens == 0 || r->n_seqs == 0 || r->pages_per_seq == 0 || (r->q && r->n_heads == 0)) return Q_ERR_INVALID_SIZE;
    if (r->kv.head_dim > 256 || (!r->seq && r->n_tokens > r->n_seqs)) return Q_ERR_INVALID_SIZE;
    if ((uint64_t)2 * r->kv.n_kv_heads + (r->q ? r->n_heads : 0) > 65535) return Q_ERR_INVALID_SIZE;
    if (r->plan)
        if (q_error_code rc = check_plan(r->plan, r->kv.head_dim)) return rc;
    const uint32_t es = size_of(r->dtype), ec = size_of(r->kv.dtype);
    if (((addr(r->k) | addr(r->v) | addr(r->q) | addr(r->q_out)) & (es - 1)) ||
        ((addr(r->pages) | addr(r->seq) | addr(r->row) | addr(r->pos)) & 3))
        return Q_ERR_MISALIGNED;
    if (!short_strides({r->k_token_stride, r->k_head_stride, r->v_token_stride, r->v_head_stride}) ||
        (r->q && !short_strides({r->q_token_stride, r->q_head_stride, r->q_out_token_stride, r->q_out_head_stride})))
        return Q_ERR_INVALID_SIZE;
    if (r->q && r->q == r->q_out && (r->q_token_stride != r->q_out_token_stride || r->q_head_stride != r->q_out_head_stride))
        return Q_ERR_ALIASING;
    if (!DevicePtrs()(r->kv.k)(r->kv.v)(r->k)(r->v)(r->q)(r->q ? r->q_out : nullptr)(r->pages)(r->seq)(r->row)(r->pos).ok)
        return Q_ERR_INVALID_ARG;
    RotateArgs a{};
    set_plan(a, r->plan, false);
    a.pos = r->pos;
    a.row = r->row;
    a.seq = r->seq;
    a.pages = r->pages;
    a.page_stride = r->kv.page_stride;
    a.row_stride = (uint32_t)r->kv.row_stride;
    a.page_rows = fast_div_of(r->kv.page_rows);
    a.n_pages = r->kv.n_pages;
    a.pages_per_seq = r->pages_per_seq;
    a.n_seqs = r->n_seqs;
    a.n_tokens = r->n_tokens;
    a.head_dim = r->kv.head_dim;
    const uint64_t hs = r->kv.head_stride;
    const bool rot = r->plan != nullptr;
    a.part[0] = rotate_rows(r->k, r->kv.k, r->k_token_stride, r->k_head_stride, 0, hs, r->kv.n_kv_heads, rot);
    a.part[1] = rotate_rows(r->v, r->kv.v, r->v_token_stride, r->v_head_stride, 0, hs, r->kv.n_kv_heads, false);
    if (r->q)
        a.part[2] = rotate_rows(r->q, r->q_out, r->q_token_stride, r->q_head_stride, r->q_out_token_stride,
                                r->q_out_head_stride, r->n_heads, rot);
    uint64_t in = align_of({addr(r->k), addr(r->v), r->k_token_stride * es, r->k_head_stride * es, r->v_token_stride * es,
                            r->v_head_stride * es});
    if (r->q)
        in = std::min(in, align_of({addr(r->q), addr(r->q_out), r->q_token_stride * es, r->q_head_stride * es,
                                    r->q_out_token_stride * es, r->q_out_head_stride * es}));
    const uint64_t to = align_of({addr(r->kv.k), addr(r->kv.v), r->kv.page_stride * ec, hs * ec, r->kv.row_stride * ec});
    uint32_t E = es == 4 && ec == 4 ? 4 : 8;
    while (E > 1 && !(vectors_fit(E, es, in, a) && vectors_fit(E, ec, to, a))) E = E == 8 ? 4 : 1;
    cudaStream_t st = (cudaStream_t)stream;
    auto go = [&](auto ti) -> cudaError_t {
        using TI = decltype(ti);
        switch (r->kv.dtype) {
            case Q_B200_F32: return launch_rotate<TI, float>(a, E, st);
            case Q_B200_F16: return launch_rotate<TI, __half>(a, E, st);
            default: return launch_rotate<TI, __nv_bfloat16>(a, E, st);
        }
    };
    switch (r->dtype) {
        case Q_B200_F32: Q_CUDA(go(float())); break;
        case Q_B200_F16: Q_CUDA(go(__half())); break;
        default: Q_CUDA(go(__nv_bfloat16())); break;
    }
    return Q_OK;
}

}  // extern "C"

// ---- attention --------------------------------------------------------------------

namespace {

enum AttnKernel { ATTN_FEW, ATTN_ROWS, ATTN_TC };
struct AttnPass {
    AttnKernel kern = ATTN_FEW;
    uint32_t mb = 1;                 // FEW: blocks of 16 vectors
    uint32_t tiles = 0, items = 0, splits = 1, parts = 1;
    bool cluster = false;            // FEW: the splits join within a cluster
    bool alternate = false;          // TC: one tile of vectors
};
struct AttnPlan {
    bool shared = false;  // a pass of its own for the prefix
    AttnPass pre, own;
    uint32_t parts = 0;   // partial results in the workspace
};

// Most rows of one running sum.  The tensor core truncates what it adds to a
// sum, 2^-24.4 of it for each product of 16 rows on tcgen05 and 2^-23.4 on
// mma.sync (a million equal values in one sum came out 0.3% and 0.15% low), so
// a sum ends after 1024 and 512 of them: 5e-5 at most, a tenth of fp16's half
// step.  Rows past that are cut into more parts, which are added in fp32.  The
// sums of fp32 caches are rounded instead, which equal values share too.
constexpr uint32_t TC_SUM_ROWS = 1024 * 16, WARP_SUM_ROWS = 512 * 16;

// CTAs on an SM that a pass is cut for: those that run there at once, by
// registers and shared memory, but for attn_rows_kernel on fp32 rows of 128,
// whose ring (131 KB) leaves room for one.  Parts for two share out better
// there: 16 x 1 tokens of 32/8 heads over 4096 + 1024 rows take 101 us and 112
// with parts for one, 8 x 5 of 64/8 heads over 4096 + 512 rows 296 and 354, 4 x
// 32 of 32/8 heads over 1024 + 512 rows 157 and 191 (1 x 64 over 2048 own rows
// alone 72 and 65).
uint32_t ctas_per_sm(const AttnPass& p) { return p.kern == ATTN_TC ? 1 : p.kern == ATTN_FEW && p.mb == 1 ? 3 : 2; }

// A pass of attn_few_kernel (up to 32 vectors) or attn_rows_kernel: the rows
// are cut until as many CTAs as `sms` run at once have work, each with at least
// two tiles, and a warp's sums end in time.  Up to 8 cuts of the own rows are
// one cluster's and leave nothing in the workspace.
AttnPass plan_pass(uint32_t vecs, uint32_t seqs, uint32_t kv_heads, uint32_t rows, uint32_t step, bool own, uint32_t sms) {
    AttnPass p;
    p.kern = vecs <= 32 ? ATTN_FEW : ATTN_ROWS;
    p.mb = vecs <= 16 ? 1 : 2;
    p.tiles = cdiv(vecs, p.kern == ATTN_FEW ? 16 * p.mb : ATTN_VECS);
    p.items = p.tiles * seqs;
    const uint64_t ctas = (uint64_t)p.items * kv_heads;
    const uint32_t most = std::max(1u, cdiv(rows, 2 * step));
    p.splits = (uint32_t)std::min<uint64_t>({std::max<uint64_t>(1, ctas_per_sm(p) * sms / ctas), most, 64});
    // the rows are shared out over four warps (FEW), or all four take each
    p.splits = std::max(p.splits, cdiv(rows, p.kern == ATTN_FEW ? 4 * WARP_SUM_ROWS : WARP_SUM_ROWS));
    if (p.kern == ATTN_FEW && own && p.splits > 1) {
        p.cluster = p.splits <= 8 || rows <= 8 * 4 * step;
        if (p.cluster) p.splits = std::min(p.splits, 8u);
    }
    p.parts = own && (p.cluster || p.splits == 1) ? 0 : p.splits;
    return p;
}

// The prefix on tcgen05: a tile of 128 vectors (two where there are more)
// per CTA, one CTA per SM, the rows cut so that `sms` SMs have one, but each
// four tiles: a shorter part costs as much to begin, and to add later, as to
// compute.
AttnPass plan_tc(uint32_t vecs, uint32_t kv_heads, uint32_t rows, uint32_t sms) {
    AttnPass p;
    p.kern = ATTN_TC;
    p.alternate = vecs <= 128;
    p.tiles = p.items = cdiv(vecs, p.alternate ? 128 : 256);
    const uint32_t ctas = p.items * kv_heads;
    p.splits = std::min({std::max(1u, sms / ctas), std::max(1u, rows / (4 * TC_ROWS)), ATTN_MAX_PARTS});
    p.splits = std::max(p.splits, cdiv(rows, p.alternate ? 2 * TC_SUM_ROWS : TC_SUM_ROWS));
    p.parts = p.splits;
    return p;
}

q_error_code check_attn(const q_b200_attn_args* r) {
    if (!known(r->kv.dtype)) return Q_ERR_INVALID_DTYPE;
    const q_b200_paged_kv& kv = r->kv;
    if (kv.n_pages == 0 || kv.page_rows == 0 || kv.page_rows > (1u << 30) || kv.n_kv_heads == 0) return Q_ERR_INVALID_SIZE;
    if (kv.head_dim != 32 && kv.head_dim != 64 && kv.head_dim != 128) return Q_ERR_INVALID_SIZE;
    if (r->n_tokens == 0 || r->n_seqs == 0 || r->n_heads == 0 || r->max_q == 0 || r->pages_per_seq == 0) return Q_ERR_INVALID_SIZE;
    if (r->n_heads % kv.n_kv_heads || kv.n_kv_heads > 65535) return Q_ERR_INVALID_SIZE;
    const uint64_t most_q = (uint64_t)r->n_seqs * r->max_q;  // bounded before it is multiplied on: three factors can pass 2^64
    if ((uint64_t)r->n_tokens * r->n_heads >= (1u << 30) || most_q >= (1u << 30) || most_q * r->n_heads >= (1u << 30))
        return Q_ERR_INVALID_SIZE;
    if ((uint64_t)r->max_len + r->max_prefix >= (1u << 30)) return Q_ERR_INVALID_SIZE;
    if ((uint64_t)r->pages_per_seq * kv.page_rows < r->max_len) return Q_ERR_INVALID_SIZE;
    return Q_OK;
}

AttnPlan plan_attn(const q_b200_attn_args* r) {
    const uint32_t G = r->n_heads / r->kv.n_kv_heads, step = r->kv.dtype == Q_B200_F32 ? 32 : 64;
    AttnPlan p;
    const uint32_t prefix = r->max_prefix;
    // A pass of its own reads the prefix once instead of once per sequence
    // (from L2 after the first); it costs a launch and its parts.
    p.shared = prefix >= 2 * step && r->n_seqs > 1;
    const uint32_t heads = r->kv.n_kv_heads, own_rows = std::max(1u, r->max_len + (p.shared ? 0 : prefix));
    auto own = [&](uint32_t sms) { return plan_pass(r->max_q * G, r->n_seqs, heads, own_rows, step, true, sms); };
    if (!p.shared) {
        p.own = own(SMS);
    } else {
        const uint32_t vecs = r->n_tokens * G;
        const bool tc = r->kv.dtype != Q_B200_F32 && r->kv.head_dim >= 64 && r->scale > 0.0f && vecs > 32;
        auto pre = [&](uint32_t sms) { return tc ? plan_tc(vecs, heads, prefix, sms) : plan_pass(vecs, 1, heads, prefix, step, false, sms); };
        // The two passes may run side by side, if the own rows' CTAs all find
        // room beside the prefix's (they wait for them before they add the
        // parts): the SMs are shared by what each pass takes, in whole sets of
        // the own rows' CTAs, so that (fp32 rows of 128 aside) none has to wait
        // for the prefix's SMs.  Or one pass follows the other and each has the
        // whole GPU.  SM microseconds as measured: 3 to 5 for a CTA's begin and
        // end; 0.9 for a tile of 128 rows on tcgen05, 1.9 for two streams'
        // vectors; 0.95 to 1.6 for a chunk (16 rows, 8 of fp32) of a warp.
        // Lengths are taken to be spread over max_len, 0.6 of it on the average.
        const AttnPass one = own(0), pt = pre(0);
        const double n_own = (double)one.items * heads, n_pre = (double)pt.items * heads;
        const double need = std::ceil(n_own / ctas_per_sm(one));
        const double chunk = 4.0 * ctas_per_sm(one) * (step / 4) / (step == 32 ? 1.6 : 0.95);
        const double t_own = n_own * (0.6 * own_rows / chunk + 5.0 / ctas_per_sm(one));
        const double t_pre = tc ? n_pre * (prefix / 128.0 * (pt.alternate ? 0.9 : 1.9) + 4.0 * SMS / (2 * n_pre))
                                : n_pre * (prefix / (4.0 * ctas_per_sm(pt) * (step / 4) / (step == 32 ? 1.6 : 0.95)) + 5.0);
        double sets = std::max(1.0, std::round(SMS * t_own / (t_own + t_pre) / need));
        while (sets > 1.0 && sets * need > SMS * 0.7) --sets;  // the prefix's CTAs are the longer ones
        // Side by side saves one begin and end, 6 us, but a set can be far more
        // than the own rows' share.  Measured, side by side and one after the
        // other, bf16, 32/8 heads of 128: 16 x 1 tokens over 4096 + 1024 rows 15.8
        // and 22.7 us, 40 x 1 24.8 and 38.1, 48 x 1 41.3 and 39.7; 16 x 4 over 16384
        // + 256 rows 39.3 and 37.6, 24 x 4 64 and 48, 32 x 4 96 and 52.
        const double left = SMS - sets * need;
        if (left >= 4.0 && std::max(t_pre / left, t_own / (sets * need)) <= 1.25 * ((t_own + t_pre) / SMS + 6.0)) {
            p.pre = pre((uint32_t)left);
            const uint32_t used = cdiv((uint64_t)p.pre.items * p.pre.splits * heads, ctas_per_sm(p.pre));
            p.own = own(std::max((uint32_t)need, used < SMS ? SMS - used : 0u));
        } else {
            p.pre = pre(SMS);
            p.own = own(SMS);
        }
    }
    p.parts = (p.shared ? p.pre.parts : 0) + p.own.parts;
    return p;
}

// Items are a grid's second dimension.
bool plan_fits(const AttnPlan& p) { return p.own.items <= 65535 && p.pre.items <= 65535; }

size_t attn_bytes(const q_b200_attn_args* r, const AttnPlan& p) {
    return (size_t)p.parts * r->n_tokens * r->n_heads * (r->kv.head_dim * 4 + 8);
}

template <typename T, int HD, int MB>
cudaError_t launch_few(PrefixArgs& a, const AttnPass& p, uint32_t kv_heads, cudaStream_t st) {
    using S = FewShape<T, HD>;
    constexpr uint32_t smem = S::smem(MB);
    if (cudaError_t e = ensure_smem_attr((const void*)attn_few_kernel<T, HD, MB>, smem)) return e;
    a.cluster = p.cluster;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.splits, p.items, kv_heads);
    cfg.blockDim = dim3(FEW_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    uint32_t n = 0;
    if (p.cluster) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = p.splits;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
    cfg.attrs = attr;
    cfg.numAttrs = n;
    g_kernel_launches.fetch_add(1, std::memory_order_relaxed);
    return cudaLaunchKernelEx(&cfg, attn_few_kernel<T, HD, MB>, a);
}

template <typename T, int HD>
cudaError_t launch_pass(PrefixArgs a, const AttnPass& p, uint32_t kv_heads, cudaStream_t st) {
    a.tiles = p.tiles;
    a.splits = p.splits;
    if constexpr (sizeof(T) == 2 && HD >= 64) {
        if (p.kern == ATTN_TC) {
            a.alternate = p.alternate;
            if (cudaError_t e = ensure_smem_attr((const void*)attn_prefix_tc_kernel<T, HD>, (int)TcShape<HD>::SMEM)) return e;
            return launch_ex(attn_prefix_tc_kernel<T, HD>, dim3(p.splits, p.items, kv_heads), dim3(TC_THREADS),
                             TcShape<HD>::SMEM, st, true, a);
        }
    }
    if (p.kern == ATTN_FEW)
        return p.mb == 1 ? launch_few<T, HD, 1>(a, p, kv_heads, st) : launch_few<T, HD, 2>(a, p, kv_heads, st);
    const size_t smem = attn_rows_smem<T, HD>();
    if (cudaError_t e = ensure_smem_attr((const void*)attn_rows_kernel<T, HD>, (int)smem)) return e;
    return launch_ex(attn_rows_kernel<T, HD>, dim3(p.splits, p.items, kv_heads), dim3(ATTN_THREADS), smem, st, true, a);
}

// The prefix's pass, then the own rows' beside its tail (programmatic
// dependent launch: a pass that is not the call's first waits for the one
// before it only when its own rows are done), which adds the prefix's parts itself unless its rows are
// in parts too: then the join adds all of them.
template <typename T, int HD>
cudaError_t launch_attn(PrefixArgs& a, const AttnPlan& p, uint32_t kv_heads, cudaStream_t st) {
    cudaError_t e = cudaSuccess;
    if (p.shared) {
        a.shared = a.first = 1;
        if ((e = launch_pass<T, HD>(a, p.pre, kv_heads, st))) return e;
    }
    a.shared = 0;
    a.first = !p.shared;
    a.with_prefix = !p.shared;
    a.part0 = p.shared ? p.pre.parts : 0u;
    a.last = p.own.parts == 0;
    a.merge = a.last ? a.part0 : 0u;
    if ((e = launch_pass<T, HD>(a, p.own, kv_heads, st)) || a.last) return e;
    a.n_parts = p.parts;
    return launch_ex(attn_join_kernel<T, HD>, dim3(cdiv((uint64_t)a.n_tokens * a.n_heads * (HD / 4), 128)), dim3(128), 0, st, true, a);
}

template <typename T>
cudaError_t launch_attn_dim(PrefixArgs& a, const AttnPlan& p, const q_b200_paged_kv& kv, cudaStream_t st) {
    if (kv.head_dim == 32) return launch_attn<T, 32>(a, p, kv.n_kv_heads, st);
    if (kv.head_dim == 64) return launch_attn<T, 64>(a, p, kv.n_kv_heads, st);
    return launch_attn<T, 128>(a, p, kv.n_kv_heads, st);
}

}  // namespace

extern "C" {

size_t q_b200_attn_work_bytes(const q_b200_attn_args* r) {
    if (!r || check_attn(r) != Q_OK) return 0;
    const AttnPlan p = plan_attn(r);
    return plan_fits(p) ? attn_bytes(r, p) : 0;
}

q_error_code q_b200_attn_prefix(const q_b200_attn_args* r, void* stream) {
    if (!r || !r->q || !r->out || !r->pages || !r->lens) return Q_ERR_INVALID_ARG;
    if (q_error_code rc = check_cache(r->kv)) return rc;
    if (q_error_code rc = check_attn(r)) return rc;
    if (r->max_prefix && (!r->prefix_pages || !r->prefix_len)) return Q_ERR_INVALID_ARG;
    if (!r->q_start && (r->max_q != 1 || r->n_tokens != r->n_seqs)) return Q_ERR_INVALID_SIZE;
    if (!std::isfinite(r->scale)) return Q_ERR_INVALID_ARG;
    if (r->q == r->out) return Q_ERR_ALIASING;
    const uint32_t es = size_of(r->kv.dtype);
    const uint64_t in = align_of({addr(r->q), addr(r->kv.k), addr(r->kv.v), r->q_token_stride * es, r->q_head_stride * es,
                                  r->kv.page_stride * es, r->kv.head_stride * es, r->kv.row_stride * es});
    const uint64_t to = align_of({addr(r->out), r->out_token_stride * es, r->out_head_stride * es});
    if (in < 16 || to < 16) return Q_ERR_MISALIGNED;
    if ((addr(r->q_start) | addr(r->pages) | addr(r->lens) | addr(r->prefix_pages) | addr(r->prefix_len)) & 3) return Q_ERR_MISALIGNED;
    const AttnPlan p = plan_attn(r);
    if (!plan_fits(p)) return Q_ERR_INVALID_SIZE;
    const size_t need = attn_bytes(r, p);
    if (need && !r->work) return Q_ERR_INVALID_ARG;
    if (need && r->work_bytes < need) return Q_ERR_INVALID_SIZE;
    if (need && (addr(r->work) & 15)) return Q_ERR_MISALIGNED;
    const bool pre = r->max_prefix > 0;
    if (!DevicePtrs()(r->kv.k)(r->kv.v)(r->q)(r->out)(r->q_start)(r->pages)(r->lens)(pre ? r->prefix_pages : nullptr)(
             pre ? r->prefix_len : nullptr)(need ? r->work : nullptr).ok)
        return Q_ERR_INVALID_ARG;
    PrefixArgs a{};
    a.q = r->q;
    a.out = r->out;
    a.k = r->kv.k;
    a.v = r->kv.v;
    a.q_token = r->q_token_stride;
    a.q_head = r->q_head_stride;
    a.o_token = r->out_token_stride;
    a.o_head = r->out_head_stride;
    a.page_stride = r->kv.page_stride;
    a.head_stride = r->kv.head_stride;
    a.row_stride = r->kv.row_stride;
    a.q_start = r->q_start;
    a.pages = r->pages;
    a.lens = r->lens;
    a.prefix_pages = pre ? r->prefix_pages : nullptr;
    a.prefix_len = pre ? r->prefix_len : nullptr;
    a.part_o = (float*)r->work;
    a.part_ml = (float2*)((float*)r->work + (size_t)p.parts * r->n_tokens * r->n_heads * r->kv.head_dim);
    a.page_rows = fast_div_of(r->kv.page_rows);
    a.group = r->n_heads / r->kv.n_kv_heads;
    a.by_group = fast_div_of(a.group);
    a.n_pages = r->kv.n_pages;
    a.pages_per_seq = r->pages_per_seq;
    a.n_tokens = r->n_tokens;
    a.n_seqs = r->n_seqs;
    a.n_heads = r->n_heads;
    a.max_q = r->max_q;
    a.max_len = r->max_len;
    a.max_prefix = r->max_prefix;
    a.c = r->scale * 1.44269504088896341f;
    cudaStream_t st = (cudaStream_t)stream;
    switch (r->kv.dtype) {
        case Q_B200_F32: Q_CUDA(launch_attn_dim<float>(a, p, r->kv, st)); break;
        case Q_B200_F16: Q_CUDA(launch_attn_dim<__half>(a, p, r->kv, st)); break;
        default: Q_CUDA(launch_attn_dim<__nv_bfloat16>(a, p, r->kv, st)); break;
    }
    return Q_OK;
}

}  // extern "C"

// ---- drafts -------------------------------------------------------------------------

namespace {

template <typename T, int KIND>
cudaError_t launch_verify(const VerifyArgs& a, uint32_t n_seqs, uint32_t CL, cudaStream_t st) {
    const void* kern = (const void*)verify_kernel<T, KIND>;
    if (CL > 8)
        if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(n_seqs * CL);
    cfg.blockDim = dim3(VER_THREADS);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = CL;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    g_kernel_launches.fetch_add(1, std::memory_order_relaxed);
    return cudaLaunchKernelEx(&cfg, verify_kernel<T, KIND>, a);
}

template <typename T>
cudaError_t launch_verify_kind(const VerifyArgs& a, int kind, uint32_t n_seqs, uint32_t CL, cudaStream_t st) {
    if (kind == VER_PROBS) return launch_verify<T, VER_PROBS>(a, n_seqs, CL, st);
    if (kind == VER_LOGITS) return launch_verify<T, VER_LOGITS>(a, n_seqs, CL, st);
    return launch_verify<T, VER_GREEDY>(a, n_seqs, CL, st);
}

}  // namespace

extern "C" {

q_error_code q_b200_verify_draft(const q_b200_verify_args* r, void* stream) {
    if (!r || !r->target || !r->uniform || !r->tokens || !r->n_tokens) return Q_ERR_INVALID_ARG;
    if (r->n_draft && !r->draft_tokens) return Q_ERR_INVALID_ARG;
    if (!known(r->dtype)) return Q_ERR_INVALID_DTYPE;
    if (r->kind > Q_B200_LOGITS) return Q_ERR_INVALID_ARG;
    if (r->n_seqs == 0 || r->vocab == 0 || r->vocab > (1u << 30) || r->n_draft > VER_MAX_DRAFT || r->n_seqs > (1u << 26))
        return Q_ERR_INVALID_SIZE;
    if (r->kind == Q_B200_LOGITS && !(r->temperature >= 0.0f && std::isfinite(r->temperature))) return Q_ERR_INVALID_ARG;
    const uint32_t es = size_of(r->dtype);
    if (((addr(r->target) | addr(r->draft)) & (es - 1)) ||
        ((addr(r->draft_tokens) | addr(r->draft_len) | addr(r->uniform) | addr(r->tokens) | addr(r->n_tokens)) & 3))
        return Q_ERR_MISALIGNED;
    // one sequence's outputs would be written over what another has yet to read
    const uint64_t S = r->n_seqs, K = r->n_draft, tb = S * (K + 1) * 4, nb = S * 4;
    for (const auto& in : {std::make_pair((const void*)r->draft_tokens, S * K * 4), std::make_pair((const void*)r->draft_len, nb),
                           std::make_pair((const void*)r->uniform, tb)})
        if (overlap(r->tokens, tb, in.first, in.second) || overlap(r->n_tokens, nb, in.first, in.second)) return Q_ERR_ALIASING;
    if (overlap(r->tokens, tb, r->n_tokens, nb)) return Q_ERR_ALIASING;
    if (!DevicePtrs()(r->target)(r->draft)(r->draft_tokens)(r->draft_len)(r->uniform)(r->tokens)(r->n_tokens).ok)
        return Q_ERR_INVALID_ARG;
    VerifyArgs a{};
    a.target = r->target;
    a.draft = r->n_draft ? r->draft : nullptr;
    a.t_seq = r->target_seq_stride;
    a.t_row = r->target_row_stride;
    a.d_seq = r->draft_seq_stride;
    a.d_row = r->draft_row_stride;
    a.draft_tokens = r->draft_tokens;
    a.draft_len = r->draft_len;
    a.uniform = r->uniform;
    a.tokens = r->tokens;
    a.n_tokens = r->n_tokens;
    a.n_draft = r->n_draft;
    a.vocab = r->vocab;
    uint64_t by = align_of({addr(r->target), a.t_seq * es, a.t_row * es});
    if (a.draft) by = std::min(by, align_of({addr(r->draft), a.d_seq * es, a.d_row * es}));
    a.vec = by >= 16 && r->vocab >= 8;
    const int kind = r->kind == Q_B200_PROBS ? VER_PROBS : r->temperature < 1e-6f ? VER_GREEDY : VER_LOGITS;
    if (kind == VER_LOGITS) {
        a.cd = 1.44269504088896340736 / (double)r->temperature;
        a.c = (float)a.cd;
    }
    // CTAs of a sequence: as many as run at once, but a warp's segment fills a
    // lane's vectors at least once; 16 of them, which not every part of the
    // GPU has room for, only for a few sequences
    const uint32_t once = ver_vecs(kind) * 32 * (16 / es) * VER_WARPS;
    uint32_t CL = r->n_seqs <= 4 ? 16 : 8;
    while (CL > 1 && ((uint64_t)r->n_seqs * CL > (uint64_t)SMS * ver_ctas(kind) || (uint64_t)(CL / 2) * once >= r->vocab)) CL /= 2;
    a.seg = (cdiv(r->vocab, (uint64_t)CL * VER_WARPS) + 7) & ~7u;
    cudaStream_t st = (cudaStream_t)stream;
    switch (r->dtype) {
        case Q_B200_F32: Q_CUDA(launch_verify_kind<float>(a, kind, r->n_seqs, CL, st)); break;
        case Q_B200_F16: Q_CUDA(launch_verify_kind<__half>(a, kind, r->n_seqs, CL, st)); break;
        default: Q_CUDA(launch_verify_kind<__nv_bfloat16>(a, kind, r->n_seqs, CL, st)); break;
    }
    return Q_OK;
}

q_error_code q_b200_batch_kv_view(q_context* ctx, uint32_t layer, q_b200_paged_kv* kv, const uint32_t** pages,
                                  uint32_t* pages_per_seq) {
    if (!ctx || !kv || !pages || !pages_per_seq) return Q_ERR_INVALID_ARG;
    DevState* s = state_of(ctx, false);
    if (!s || !s->batch.kv || !s->batch.d_pages) return Q_ERR_INVALID_ARG;  // not a batch with paged caches
    if (layer >= s->cfg.n_layers) return Q_ERR_INVALID_SIZE;
    if (q_error_code rc = batch_sync_pages(s)) return rc;
    const BatchState& b = s->batch;
    const uint64_t head = (uint64_t)b.page_rows * 2 * s->hd;
    *kv = q_b200_paged_kv{};
    kv->k = b.kv + layer * s->tp.nkv * head;
    kv->v = b.kv + layer * s->tp.nkv * head + s->hd;
    kv->page_stride = (uint64_t)s->cfg.n_layers * s->tp.nkv * head;
    kv->head_stride = head;
    kv->row_stride = 2 * s->hd;
    kv->n_pages = b.n_pages;
    kv->page_rows = b.page_rows;
    kv->n_kv_heads = s->tp.nkv;
    kv->head_dim = s->hd;
    kv->dtype = Q_B200_F32;
    *pages = b.d_pages;
    *pages_per_seq = b.pages_per_seq;
    return Q_OK;
}

}  // extern "C"
