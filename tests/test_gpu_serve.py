"""The serving operators on the B200 against plain forms in 64 bits, at the sizes, masks and layouts where they can go wrong.

Tolerances count roundings.  H = finfo(type).eps / 2 is the largest relative error of one rounding to a type's
normal numbers; below them the step no longer shrinks, and a rounding is off by half of the smallest subnormal at most (fp16: 2^-25
below 2^-14; of no account in fp32 and bf16).

rotation: the angle's fraction of a turn is rounded to fp32 (2^-25 of a turn at most: 2^-25 * 2 pi < 2^-22 rad) and sine and
cosine are good to 2^-22 (2 ulp), so each product is off by 2^-21 of |a| or |b| with its own rounding, and the result once more
by H: |y - y64| <= gain * 2^-20 (|a| + |b|) + H |y|.

attention: with Y = scale * sum |q_i k_i| (the largest over the rows a vector sees) and A = sum p|v| / sum p, a score is off by at
most 2^-20 Y (tf32 halves drop 2^-22 of an operand's product three times over; sums of at most 128 terms are folded or truncated
at 2^-23; one product by the scale), an exponential by that and 2^-22, so numerator and denominator together shift the result by
2 (2^-20 Y + 2^-21) A, and sums over parts and rows by another 2^-18 A at most (truncation at 2^-23 of up to 32 running sums).  P
in 16 bits adds H A in the numerator and H |o| in the denominator, the result's own rounding H |o|.

verify: whole numbers, equal.
"""
import ctypes as C
import math

import numpy as np
import pytest

import qorus_b200 as Q

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = {"f32": (torch.float32, Q.Q_B200_F32), "f16": (torch.float16, Q.Q_B200_F16), "bf16": (torch.bfloat16, Q.Q_B200_BF16)}


def half_step(dtype):
    return torch.finfo(TYPES[dtype][0]).eps / 2


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(g, *shape, dtype="f32"):
    return torch.randn(shape, generator=g, device="cuda").to(TYPES[dtype][0])


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def stream():
    return torch.cuda.current_stream().cuda_stream


def scale_of(kind):
    return Q.q_b200_rope_scale({"plain": 0, "linear": 1, "banded": 2, "yarn": 3}[kind], 0, 8.0, 1.0, 32.0 if kind == "yarn" else 4.0,
                               8192.0, 0.0)


def make_plan(rot, layout="half", kind="plain", base=500000.0):
    p = Q.q_b200_rope_plan()
    Q.check(Q.lib.q_b200_rope_plan_init(C.byref(p), rot, int(layout == "half"), base, C.byref(scale_of(kind))), "plan")
    return p


def turn64(x, pos, p, back=False):
    """Rotation by a plan's turns in 64 bits (the plan itself is tested against the formulas without a GPU)."""
    rot, half = p.rot_dim, p.layout == Q.Q_B200_ROPE_HALF
    w = torch.tensor(list(p.turns[: rot // 2]), dtype=torch.float64, device="cuda") * (2 * math.pi)
    ang = (pos.double()[:, None] * w)[:, None]
    c, s = ang.cos() * p.gain, ang.sin() * (-p.gain if back else p.gain)
    y = x.double().clone()
    ia = torch.arange(rot // 2, device="cuda") * (1 if half else 2)
    ib = ia + (rot // 2 if half else 1)
    a, b = y[..., ia].clone(), y[..., ib].clone()
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    room = torch.zeros_like(y)
    room[..., ia] = room[..., ib] = (a.abs() + b.abs()) * p.gain * 2.0**-20
    return y, room


def do_rope(x, out, pos, p, back=False, dtype="f32", on=None):
    a = Q.q_b200_rope_args(x.data_ptr(), out.data_ptr(), pos.data_ptr(), C.addressof(p), x.stride(0), x.stride(1), out.stride(0),
                           out.stride(1), x.shape[0], x.shape[1], x.shape[2], TYPES[dtype][1], int(back), 0)
    Q.check(Q.lib.q_b200_rope(C.byref(a), stream() if on is None else on), "q_b200_rope")


def within(got, want, room, dtype):
    err = (got.double() - want).abs()
    lim = room + half_step(dtype) * want.abs() + torch.finfo(TYPES[dtype][0]).smallest_normal * half_step(dtype)
    bad = ~(err <= lim)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside; worst {float((err - lim)[bad].max()):.3e} over {float(lim[bad].max()):.3e}"


# ---- rotation ---------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,heads,dim,rot,kind,far", [
    (1, 1, 2, 2, "plain", 10), (1, 32, 128, 128, "plain", 8192), (3, 5, 80, 40, "linear", 1000), (7, 3, 33, 18, "plain", 500),
    (129, 8, 64, 32, "yarn", 1 << 20), (257, 40, 128, 96, "banded", 1 << 20), (2, 2, 256, 256, "yarn", (1 << 31) - 1),
    (5000, 9, 64, 64, "plain", 131072)])
def test_rope(dtype, layout, tokens, heads, dim, rot, kind, far):
    g, p = gen(tokens + dim), make_plan(rot, layout, kind)
    x = normal(g, tokens, heads, dim, dtype=dtype)
    pos = torch.randint(-far, far, (tokens,), generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
    pos[0] = far - 1
    out = torch.full_like(x, 7.0)
    do_rope(x, out, pos, p, dtype=dtype)
    want, room = turn64(x, pos, p)
    within(out, want, room, dtype)
    assert torch.equal(out[..., rot:], x[..., rot:])
    # the way back, in place, and out of rows that lie inside a wider buffer
    wide = torch.zeros(tokens, heads + 3, dim + 7, dtype=x.dtype, device="cuda")
    view = wide[:, 2:2 + heads, :dim]
    view.copy_(x)
    do_rope(view, view, pos, p, back=True, dtype=dtype)
    want, room = turn64(x, pos, p, back=True)
    within(view, want, room, dtype)
    assert wide[:, :2].abs().max() == 0 and wide[:, 2 + heads:].abs().max() == 0 and wide[..., dim:].abs().max() == 0


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope_transpose_is_the_gradient(layout):
    # <y, R x> = <R^T y, x>, and a difference of the linear map is the map of the difference
    g, p = gen(3), make_plan(48, layout, "yarn")
    x, y = normal(g, 50, 4, 64), normal(g, 50, 4, 64)
    pos = torch.randint(0, 100000, (50,), generator=g, device="cuda", dtype=torch.int32)
    rx, ry, rd = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    do_rope(x, rx, pos, p)
    do_rope(y, ry, pos, p, back=True)
    a, b = (y.double() * rx.double()).sum(), (ry.double() * x.double()).sum()
    # 12800 products, each off by 2^-20 (|a| + |b|) * gain at most
    room = p.gain * 2.0**-20 * 4 * float((x.double().abs().sum() + y.double().abs().sum()) * max(x.abs().max(), y.abs().max()))
    assert abs(float(a - b)) <= room
    do_rope(x + y, rd, pos, p)
    ry2 = torch.empty_like(x)
    do_rope(y, ry2, pos, p)
    _, r1 = turn64(x + y, pos, p)
    _, r2 = turn64(x, pos, p)
    _, r3 = turn64(y, pos, p)
    assert ((rd.double() - rx.double() - ry2.double()).abs() <= r1 + r2 + r3 + 2.0**-22 * (x.abs() + y.abs()).double()).all()


def test_rope_matches_the_host_call_at_small_positions():
    g, p = gen(5), make_plan(128, "interleaved")
    x = normal(g, 1, 1, 128)
    out = torch.empty_like(x)
    do_rope(x, out, ints([37]), p)
    ang = (37.0 * np.array(p.turns[:64]) * 2 * math.pi).repeat(2)
    hx, hc, hs, ho = (Q.aligned_empty(128) for _ in range(4))
    hx[:], hc[:], hs[:] = x.cpu().numpy().ravel(), np.cos(ang), np.sin(ang)
    Q.check(Q.lib.q_rope_f32_avx2(Q.ptr(hx), Q.ptr(hc), Q.ptr(hs), Q.ptr(ho), 128), "q_rope_f32_avx2")
    np.testing.assert_allclose(out.cpu().numpy().ravel(), ho, atol=2.0**-20 * 2 * float(x.abs().max()), rtol=0)


# ---- paged append -----------------------------------------------------------------------------------------------------


def new_pool(g, pages, layers, kv_heads, rows, dim, dtype):
    pool = normal(g, pages, layers, kv_heads, rows, 2 * dim, dtype=dtype)
    return pool, pool[:, -1, ..., :dim], pool[:, -1, ..., dim:]


def cache_of(keys, values, dtype):  # [page][head][row][dim] views of equal strides
    return Q.q_b200_paged_kv(keys.data_ptr(), values.data_ptr(), keys.stride(0), keys.stride(1), keys.stride(2), keys.shape[0],
                             keys.shape[2], keys.shape[1], keys.shape[3], TYPES[dtype][1], 0)


def do_append(keys, values, cache, k, v, pages, seq, row, pos, p, dtype, q=None, q_out=None):
    a = Q.q_b200_append_args(cache_of(keys, values, cache), k.data_ptr(), v.data_ptr(), None if q is None else q.data_ptr(),
                             None if q is None else q_out.data_ptr(), k.stride(0), k.stride(1), v.stride(0), v.stride(1),
                             0 if q is None else q.stride(0), 0 if q is None else q.stride(1), 0 if q is None else q_out.stride(0),
                             0 if q is None else q_out.stride(1), pages.data_ptr(), None if seq is None else seq.data_ptr(),
                             row.data_ptr(), None if pos is None else pos.data_ptr(), C.addressof(p) if p else None, k.shape[0],
                             pages.shape[0], pages.shape[1], 0 if q is None else q.shape[1], TYPES[dtype][1], 0)
    Q.check(Q.lib.q_b200_kv_append(C.byref(a), stream()), "q_b200_kv_append")


@pytest.mark.parametrize("dtype,cache", [("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16"), ("bf16", "f32"), ("f16", "f16"),
                                         ("f32", "f16"), ("f16", "bf16")])
@pytest.mark.parametrize("tokens,seqs,heads,kv_heads,dim,rot,page_rows,layout", [
    (1, 1, 4, 1, 64, 64, 1, "half"), (37, 5, 8, 2, 128, 64, 17, "interleaved"), (300, 3, 0, 3, 32, 32, 48, "half"),
    (16, 16, 32, 8, 128, 0, 32, "half"), (41, 4, 6, 3, 24, 14, 5, "interleaved"), (6000, 64, 32, 8, 64, 64, 16, "half")])
def test_append(dtype, cache, tokens, seqs, heads, kv_heads, dim, rot, page_rows, layout):
    g, p = gen(tokens), make_plan(rot, layout, "banded") if rot else None
    rows = -(-tokens // seqs) + 3
    per = -(-rows // page_rows)
    pool, keys, values = new_pool(g, seqs * per + 2, 2, kv_heads, page_rows, dim, cache)
    before = pool.clone()
    pages = torch.randperm(seqs * per + 2, generator=g, device="cuda")[: seqs * per].to(torch.int32).view(seqs, per)
    t = torch.arange(tokens, device="cuda")
    seq, row = (t % seqs).to(torch.int32), (t // seqs + 2).to(torch.int32)
    if tokens > 4:
        row[3] = -1
        row[tokens // 2] = -5
    pos = row * 3 + 100
    qkv = normal(g, tokens, (heads + 2 * kv_heads) * dim, dtype=dtype)
    q = qkv[:, : heads * dim].view(tokens, heads, dim)
    k = qkv[:, heads * dim: (heads + kv_heads) * dim].view(tokens, kv_heads, dim)
    v = qkv[:, (heads + kv_heads) * dim:].view(tokens, kv_heads, dim)
    q_out = torch.full((tokens, max(1, heads), dim), 9.0, dtype=q.dtype, device="cuda")
    do_append(keys, values, cache, k, v, pages, seq, row, pos, p, dtype, q if heads else None, q_out)
    live = row >= 0
    page = pages[seq.long()[live], row.long()[live] // page_rows].long()
    at = (page, row.long()[live] % page_rows)
    want, room = turn64(k, pos, p) if p else (k.double(), torch.zeros_like(k.double()))
    within(keys.permute(0, 2, 1, 3)[at], want[live], room[live], cache)
    assert torch.equal(values.permute(0, 2, 1, 3)[at], v[live].to(TYPES[cache][0]))
    if heads:
        want, room = turn64(q, pos, p) if p else (q.double(), torch.zeros_like(q.double()))
        within(q_out[live], want[live], room[live], dtype)
        assert (q_out[~live] == 9.0).all()
    # nothing else moved
    now = pool.clone()
    for x in (keys, values):
        x.permute(0, 2, 1, 3)[at] = 0
    rest = before.clone()
    rest[:, -1, ..., :dim].permute(0, 2, 1, 3)[at] = 0
    rest[:, -1, ..., dim:].permute(0, 2, 1, 3)[at] = 0
    assert torch.equal(pool, rest) and not torch.equal(now, rest)
    assert Q.lib.q_b200_device_status() == 0


def test_append_turns_queries_in_place():
    g, p = gen(9), make_plan(64, "interleaved")
    pool, keys, values = new_pool(g, 4, 1, 2, 8, 64, "bf16")
    qkv = normal(g, 4, 8, 64, dtype="bf16")
    q, was, row = qkv[:, :4], qkv[:, :4].clone(), ints([7, -1, 3, 0])
    do_append(keys, values, "bf16", qkv[:, 4:6], qkv[:, 6:], ints([[0], [1], [2], [3]]), None, row, None, p, "bf16", q, q)
    want, room = turn64(was, row, p)
    within(q[[0, 2, 3]], want[[0, 2, 3]], room[[0, 2, 3]], "bf16")
    assert torch.equal(q[1], was[1])


def test_append_without_sequence_and_position_lists():
    g, p = gen(1), make_plan(32)
    pool, keys, values = new_pool(g, 6, 1, 2, 4, 32, "f32")
    pages, row = ints([[5], [0], [3]]), ints([1, 3, 0])
    k, v = normal(g, 3, 2, 32), normal(g, 3, 2, 32)
    do_append(keys, values, "f32", k, v, pages, None, row, None, p, "f32")
    want, room = turn64(k, row, p)
    at = (torch.tensor([5, 0, 3], device="cuda"), row.long())
    within(keys.permute(0, 2, 1, 3)[at], want, room, "f32")
    assert torch.equal(values.permute(0, 2, 1, 3)[at], v)


def test_append_skips_what_names_no_page():
    g = gen(2)
    pool, keys, values = new_pool(g, 3, 1, 1, 4, 32, "f32")
    before = pool.clone()
    pages, seq, row = ints([[0, 3], [-1, 2]]), ints([0, 1, 2, 0, 1]), ints([5, 0, 1, 8, 6])
    k, v = normal(g, 5, 1, 32), normal(g, 5, 1, 32)
    do_append(keys, values, "f32", k, v, pages, seq, row, None, None, "f32")  # pages 3 and -1, sequence 2, row 8 of 8
    assert Q.lib.q_b200_device_status() == 4 and Q.lib.q_b200_device_status() == 0
    assert torch.equal(keys[2, 0, 2], k[4, 0]) and torch.equal(values[2, 0, 2], v[4, 0])
    keys[2, 0, 2] = before[2, 0, 0, 2, :32]
    values[2, 0, 2] = before[2, 0, 0, 2, 32:]
    assert torch.equal(pool, before)


# ---- attention ----------------------------------------------------------------------------------------------------------


class Batch:
    """A paged cache, new tokens and their 64-bit result.  Every row that nobody sees is NaN."""

    def __init__(self, seed, dtype, heads, kv_heads, dim, page_rows, prefix, rows, new, pad=0, layers=2, split_kv=False, poison=True,
                 room_rows=0):
        g = gen(seed)
        self.dtype, self.heads, self.dim, self.prefix, self.rows, self.new = dtype, heads, dim, prefix, rows, new
        B, R = len(rows), page_rows
        self.per, shared = max(1, -(-(max(rows) + room_rows) // R)), -(-prefix // R)
        n = B * self.per + shared + 1
        if split_kv:  # two pools [page][row][head][dim]
            self.keys, self.values = (normal(g, n, R, kv_heads, dim, dtype=dtype).permute(0, 2, 1, 3) for _ in range(2))
        else:
            self.pool, self.keys, self.values = new_pool(g, n, layers, kv_heads, R, dim, dtype)
        ids = torch.randperm(n, generator=g, device="cuda").to(torch.int32)
        self.prefix_pages, self.pages = ids[:shared].contiguous(), ids[shared: shared + B * self.per].view(B, self.per).contiguous()
        if poison:
            for x in (self.keys, self.values):
                x[ids[-1].long()] = math.nan
                if prefix % R:
                    x[self.prefix_pages[-1].long(), :, prefix % R:] = math.inf
                for b in range(B):
                    for j in range(self.per):
                        x[self.pages[b, j].long(), :, min(R, max(0, rows[b] - j * R)):] = math.nan
        T = sum(new)
        qkv = normal(g, T + pad, heads + 2, dim, dtype=dtype) * 2
        self.q = qkv[:, 1: heads + 1]
        self.out = torch.full((T + pad, heads, dim), 5.0, dtype=TYPES[dtype][0], device="cuda")
        self.start = ints(np.concatenate([[0], np.cumsum(new)]).tolist())
        self.lens, self.prefix_len = ints(rows), ints([prefix])
        self.tokens, self.pad = T, pad

    def args(self, max_len=None, max_prefix=None, work=None):
        q, o = self.q, self.out
        one = max(self.new) == 1 and min(self.new) == 1 and self.pad == 0
        a = Q.q_b200_attn_args(cache_of(self.keys, self.values, self.dtype), q.data_ptr(), o.data_ptr(), q.stride(0), q.stride(1),
                               o.stride(0), o.stride(1), None if one else self.start.data_ptr(), self.pages.data_ptr(), self.lens.data_ptr(),
                               self.prefix_pages.data_ptr() if self.prefix else None, self.prefix_len.data_ptr() if self.prefix else None,
                               None, 0, q.shape[0], len(self.rows), self.heads, self.per, max(max(self.new), 1),
                               max(self.rows) if max_len is None else max_len, self.prefix if max_prefix is None else max_prefix,
                               1 / math.sqrt(self.dim))
        need = Q.lib.q_b200_attn_work_bytes(C.byref(a))
        self.work = torch.full((max(16, need),), 0xFF, dtype=torch.uint8, device="cuda") if work is None else work
        a.work, a.work_bytes = self.work.data_ptr(), self.work.numel()
        return a

    def call(self, **kw):
        a = self.args(**kw)
        Q.check(Q.lib.q_b200_attn_prefix(C.byref(a), stream()), "q_b200_attn_prefix")

    def want(self):
        """(result, room) of every token, without those of no sequence."""
        G, outs, rooms = self.heads // self.keys.shape[1], [], []
        R = self.keys.shape[2]
        flat = lambda x, p: x[p.long()].transpose(1, 2).reshape(-1, x.shape[1], self.dim).double()  # noqa: E731
        at = 0
        for b, (L, n) in enumerate(zip(self.rows, self.new)):
            ks = torch.cat([flat(self.keys, self.prefix_pages)[: self.prefix], flat(self.keys, self.pages[b])[:L]])
            vs = torch.cat([flat(self.values, self.prefix_pages)[: self.prefix], flat(self.values, self.pages[b])[:L]])
            for i in range(n):
                m = self.prefix + max(0, L - n + 1 + i)
                k, v = ks[:m].repeat_interleave(G, 1), vs[:m].repeat_interleave(G, 1)
                q = self.q[at].double()
                y = torch.einsum("hd,lhd->hl", q, k) / math.sqrt(self.dim)
                p = torch.softmax(y, -1)
                o = torch.einsum("hl,lhd->hd", p, v)
                A = torch.einsum("hl,lhd->hd", p, v.abs())
                Y = (torch.einsum("hd,lhd->hl", q.abs(), k.abs()) / math.sqrt(self.dim)).amax(-1, keepdim=True) if m else torch.zeros_like(o)
                room = A * (2 * (2.0**-20 * Y + 2.0**-21) + 2.0**-18)
                if self.dtype != "f32":
                    room = room + half_step(self.dtype) * (A + o.abs())
                outs.append(o)
                rooms.append(room)
                at += 1
        return torch.stack(outs), torch.stack(rooms)

    def check(self):
        want, room = self.want()
        within(self.out[: self.tokens], want, room, self.dtype)
        assert (self.out[self.tokens:] == 5.0).all()
        assert Q.lib.q_b200_device_status() == 0


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim,page_rows,prefix,rows,new", [
    (1, 1, 32, 1, 0, [1], [1]),                                   # one row
    (4, 1, 64, 16, 0, [0, 5, 64, 65], [1, 1, 1, 1]),              # a sequence without a row: zeros
    (8, 2, 128, 32, 1, [0, 1, 31, 32, 33], [1] * 5),              # a prefix of one row
    (8, 8, 128, 48, 700, [100, 1, 257], [1] * 3),                 # heads that share nothing
    (7, 1, 64, 17, 129, [40, 3], [1, 1]),                         # an odd group, odd pages
    (32, 4, 32, 64, 1000, [600] * 9, [1] * 9),
    (16, 2, 128, 16, 333, [9, 70, 0, 5, 8], [5, 3, 2, 1, 8]),     # drafts; rows behind the newest token's, and none at all
    (6, 2, 64, 128, 64, [200, 130], [130, 33]),                   # chunks of a prompt
    (4, 4, 128, 7, 0, [50, 3], [50, 5]),                          # a prompt from its first token; early tokens see nothing
    (8, 1, 128, 64, 5000, [1, 2, 3], [1, 1, 1]),
    (64, 8, 128, 64, 2048, [100] * 17, [1] * 17),
    (8, 2, 128, 16, 100, [50], [1]),                              # one sequence: its prefix and own rows in one pass,
    (8, 2, 64, 32, 96, [700], [3]),                               # the own rows in step with the pages and not
    (48, 1, 64, 16, 33, [20], [1]),
    (40, 1, 128, 32, 600, [40, 8], [2, 1]),
])
def test_attn(dtype, heads, kv_heads, dim, page_rows, prefix, rows, new):
    b = Batch(len(rows) + dim, dtype, heads, kv_heads, dim, page_rows, prefix, rows, new, pad=3 if max(new) > 1 else 0)
    b.call()
    b.check()
    first = b.out.clone()
    b.out.fill_(5.0)
    b.call()
    assert torch.equal(first, b.out)  # the same bits on every run


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attn_other_layout_and_loose_bounds(dtype):
    b = Batch(8, dtype, 8, 2, 64, 16, 100, [50, 7, 1], [2, 1, 1], split_kv=True, room_rows=4000)
    b.prefix_pages = torch.cat([b.prefix_pages, torch.full((60,), -1, dtype=torch.int32, device="cuda")])  # never read
    prefix, b.prefix_pages_all = b.prefix, b.prefix_pages
    b.call(max_len=4000, max_prefix=1000)
    b.prefix_pages = b.prefix_pages_all[: -(-prefix // 16)]
    b.check()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("prefix", [0, 200])
def test_attn_newer_rows_do_not_reach_older_tokens(dtype, value, prefix):
    # the last two new tokens' rows hold no numbers: the tokens before them are as without them, those that see them are not
    b = Batch(4, dtype, 8, 2, 64, 16, prefix, [90, 8], [6, 5], poison=False)
    b.call()
    clean = b.out.clone()
    want, room = b.want()
    for x in (b.keys, b.values):
        for r in (88, 89):
            x[b.pages[0, r // 16].long(), :, r % 16] = value
    b.values[b.pages[1, 7 // 16].long(), :, 7 % 16] = value
    b.out.fill_(5.0)
    b.call()
    assert torch.equal(b.out[:4], clean[:4]) and torch.equal(b.out[6:10], clean[6:10])
    assert not torch.isfinite(b.out[4:6].float()).any() and not torch.isfinite(b.out[10].float()).any()
    within(clean, want, room, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim,prefix,seqs", [
    (8, 2, 64, 200, 3),     # few vectors of a KV head: up to 16,
    (24, 2, 128, 200, 2),   # up to 32,
    (32, 2, 64, 300, 5),    # up to 128,
    (64, 2, 128, 300, 9),   # and more
    (64, 2, 32, 130, 4)])
def test_attn_seen_rows_that_are_no_numbers(dtype, heads, kv_heads, dim, prefix, seqs):
    # wherever in a tile the row lies and whatever bits the NaN has, all that see it get no finite number and nobody else notices
    b = Batch(dim + seqs, dtype, heads, kv_heads, dim, 16, prefix, [20 + i for i in range(seqs)], [1] * seqs, poison=False)
    b.q[..., 0] = b.q[..., 0].abs() + 0.5  # an infinite key's score is +inf
    bits, tops = (torch.int32, (0x7F800000, 0x7FC00000, 0x7FFFFFFF, -1)) if dtype == "f32" else (
        torch.int16, (0x7C00 if dtype == "f16" else 0x7F80, 0x7FC0 if dtype == "bf16" else 0x7E00, 0x7FFF, -1))
    b.call()
    clean = b.out.clone()
    G = heads // kv_heads
    for i, r in enumerate([0, 1, 2, 3, 4, 5, 6, 7, 30, 63, 64, 126, 127, 129]):
        for x, outs in ((b.keys, slice(None)), (b.values, slice(0, 1))):
            page = x[b.prefix_pages[r // 16].long()]  # a view
            old = page[0, r % 16, 0].clone()
            page[0, r % 16, :1].view(bits).fill_(tops[i % 4])
            b.call()
            page[0, r % 16, 0] = old
            assert not torch.isfinite(b.out[:, :G, outs].float()).any(), (r, tops[i % 4])
            same = b.out.clone()
            same[:, :G, outs] = clean[:, :G, outs]
            assert torch.equal(same, clean)


def test_attn_scores_of_the_types_lowest_value():
    # keys that push every score far down, or all of them to the same value, leave the weights as they are in 64 bits
    b = Batch(6, "bf16", 4, 2, 64, 16, 65, [20, 3], [1, 1], poison=False)
    b.keys.copy_(torch.full_like(b.keys, -300.0))
    b.q.copy_(b.q.abs())
    b.call()
    want, _ = b.want()
    A = b.values.double().abs().max()
    assert ((b.out.double() - want).abs() <= half_step("bf16") * (2 * want.abs() + A) + 2.0**-16 * A).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim,prefix,seqs", [
    (8, 2, 64, 700, 3), (16, 2, 128, 1300, 5), (16, 1, 128, 4000, 9), (32, 2, 64, 2500, 20), (64, 1, 128, 1000, 9), (8, 1, 32, 900, 40)])
def test_attn_scores_that_grow_along_the_rows(dtype, heads, kv_heads, dim, prefix, seqs):
    # the running maximum has to move again and again, everywhere at another row: up to 16 exp2 units a tile, down, and up
    b = Batch(dim + prefix, dtype, heads, kv_heads, dim, 16, prefix, [40 + 7 * i for i in range(seqs)], [1] * seqs, poison=False)
    ramp = torch.rand(b.keys.shape[:3], generator=gen(1), device="cuda") * 2
    for i, pg in enumerate(b.prefix_pages.tolist()):
        ramp[pg] += 6.0 * (i * 16 / prefix)
    b.keys.mul_(ramp[..., None].to(b.keys.dtype))
    b.call()
    b.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("scale", [-0.3, 0.0])
def test_attn_scales_that_are_not_positive(dtype, scale):
    b = Batch(14, dtype, 16, 2, 64, 16, 300, [50, 20, 9, 9, 9], [1] * 5, poison=False)
    a = b.args()
    a.scale = scale
    b.work = torch.empty(max(16, Q.lib.q_b200_attn_work_bytes(C.byref(a))), dtype=torch.uint8, device="cuda")
    a.work, a.work_bytes = b.work.data_ptr(), b.work.numel()
    Q.check(Q.lib.q_b200_attn_prefix(C.byref(a), stream()), "attn")
    b.q.mul_(scale * math.sqrt(64))  # the reference's scale is 1 / sqrt(dim)
    want, room = b.want()
    within(b.out, want, room + (half_step(dtype) * 8 if dtype != "f32" else 0.0), dtype)  # q rounded again: scores off by H Y, Y < 4


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [32, 128])
@pytest.mark.parametrize("prefix,rows", [(0, [30, 5, 1, 9]), (1, [0, 0, 0, 0]), (129, [7, 0, 300, 2]), (0, [0, 0, 0, 0])])
def test_attn_lengths_far_below_their_bounds(dtype, dim, prefix, rows):
    # a plan for 5000 rows of prefix and 600 own ones meets nearly none, or none: parts without a row
    b = Batch(15, dtype, 16, 1, dim, 16, 5000, [600] * 4, [1] * 4, poison=False)
    b.lens.copy_(ints(rows))
    b.prefix_len.copy_(ints([prefix]))
    b.out.fill_(5.0)
    b.call()
    b.rows, b.prefix, pages = rows, prefix, b.prefix_pages
    b.prefix_pages = pages[: -(-prefix // 16)]
    b.check()


def test_attn_one_token_at_every_length():
    # the row count passes every boundary of pages, chunks and parts; one bound for all, as in a captured graph
    for dtype, dim in (("bf16", 128), ("f32", 64)):
        b = Batch(16, dtype, 8, 2, dim, 17, 0, [1], [1], poison=False, room_rows=400)
        for n in list(range(0, 70)) + [127, 128, 129, 255, 256, 257, 399, 400]:
            b.rows = [n]
            b.lens.copy_(ints([n]))
            b.call(max_len=400)
            b.check()


def test_attn_bad_pages_and_lengths_are_skipped():
    b = Batch(9, "f32", 4, 2, 64, 16, 64, [40, 30], [1, 1], poison=False)
    good = b.args()
    b.call()
    clean = b.out.clone()
    b.pages[1, 1] = b.keys.shape[0]  # behind the pool
    b.call()
    assert Q.lib.q_b200_device_status() == 4
    assert torch.equal(b.out[0], clean[0]) and torch.isfinite(b.out).all()
    b.pages[1, 1] = -1
    b.lens[0] = 1000  # above max_len
    b.prefix_len[0] = 5000
    b.work = None
    b.call()
    assert Q.lib.q_b200_device_status() == 4 and Q.lib.q_b200_device_status() == 0
    assert good.n_seqs == 2
    c = Batch(9, "bf16", 4, 2, 64, 16, 64, [40, 30], [3, 3], pad=2)
    c.start.copy_(ints([0, 5, 900]))  # more than max_q, more than there are
    c.call()
    assert Q.lib.q_b200_device_status() == 4


def test_attn_in_graphs_and_streams():
    # two captured graphs with a workspace each, replayed on two streams at once, at lengths that grew since the capture
    bs = [Batch(20 + i, "bf16", 8, 2, 128, 16, 300, [40, 30, 9], [1, 1, 1], poison=False, room_rows=100) for i in range(2)]
    graphs, streams = [], [torch.cuda.Stream() for _ in bs]
    for b in bs:
        b.call(max_len=140)
    torch.cuda.synchronize()
    for b, s in zip(bs, streams):
        b.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(b.graph, stream=s):
            b.call(max_len=140)
        graphs.append(b.graph)
    for step in range(3):
        for b in bs:
            b.rows = [r + 7 for r in b.rows]
            b.lens.copy_(ints(b.rows))
            b.out.fill_(5.0)
        torch.cuda.synchronize()
        for b, s in zip(bs, streams):
            with torch.cuda.stream(s):
                b.graph.replay()
        torch.cuda.synchronize()
        for b in bs:
            b.check()


def test_attn_far_pages():
    # page offsets past 2^32 elements
    free, _ = torch.cuda.mem_get_info()
    R, H, D = 1024, 8, 128
    pages = (1 << 32) // (R * H * 2 * D) + 40
    if free < pages * R * H * 2 * D * 2 + (4 << 30):
        pytest.skip("not enough memory")
    pool = torch.empty(pages, 1, H, R, 2 * D, dtype=torch.bfloat16, device="cuda")
    b = Batch(11, "bf16", 16, H, D, R, 1500, [700, 1030], [1, 1], poison=False)
    last = pages - b.keys.shape[0]
    pool[last:] = b.pool[:, -1:]
    want, room = b.want()
    b.pool, b.keys, b.values = pool, pool[:, 0, ..., :D], pool[:, 0, ..., D:]
    b.pages, b.prefix_pages = b.pages + last, b.prefix_pages + last
    b.call()
    within(b.out, want, room, "bf16")
    k, v = normal(gen(1), 2, H, D, dtype="bf16"), normal(gen(2), 2, H, D, dtype="bf16")
    do_append(b.keys, b.values, "bf16", k, v, b.pages, None, ints([699, 1029]), None, None, "bf16")
    assert torch.equal(b.keys[b.pages[1, 1].long(), :, 5], k[1]) and torch.equal(b.values[b.pages[0, 0].long(), :, 699], v[0])


def test_attn_on_a_contexts_own_pages(tmp_path):
    # the batched decode's paged caches, written through the framework's calls, seen through the view
    cfg = Q.config(vocab=259, dim=256, hidden=512, layers=2, heads=8, kv_heads=2, max_seq=256)
    Q.write_model(str(tmp_path / "m.qorus"), cfg, seed=0, threads=1)
    m = Q.Model(str(tmp_path / "m.qorus"))
    Q.check(Q.lib.q_b200_batch_init_paged(C.byref(m.ctx), C.byref(m.model), 2, 128, 4), "batch_init_paged")
    kv, pages, per = Q.q_b200_paged_kv(), C.c_void_p(), C.c_uint32()
    view = lambda layer: Q.lib.q_b200_batch_kv_view(C.byref(m.ctx), layer, C.byref(kv), C.byref(pages), C.byref(per))  # noqa: E731
    assert view(2) == -15
    host = np.random.default_rng(0).standard_normal((2, 2, 2, 256, 64), dtype=np.float32)  # [seq][layer][head][row][K|V]
    rows = [200, 77]
    for b in range(2):
        for l in range(2):
            for h in range(2):
                part = np.ascontiguousarray(host[b, l, h, : rows[b]])
                Q.check(Q.lib.q_b200_batch_kv_write(C.byref(m.ctx), b, (l * 2 + h) * 256 * 64 * 4, Q.ptr(part), part.nbytes), "kv_write")
    torch.cuda.synchronize()
    for l in range(2):
        Q.check(view(l), "view")
        assert (kv.page_rows, kv.n_kv_heads, kv.head_dim, kv.n_pages, per.value) == (128, 2, 32, 4, 2)
        q, out, lens = normal(gen(l), 2, 8, 32), torch.zeros(2, 8, 32, device="cuda"), ints(rows)
        a = Q.q_b200_attn_args(kv, q.data_ptr(), out.data_ptr(), 256, 32, 256, 32, None, pages, lens.data_ptr(), None, None, None, 0,
                               2, 2, 8, per.value, 1, 256, 0, 1 / math.sqrt(32))
        work = torch.empty(max(16, Q.lib.q_b200_attn_work_bytes(C.byref(a))), dtype=torch.uint8, device="cuda")
        a.work, a.work_bytes = work.data_ptr(), work.numel()
        torch.cuda.synchronize()
        Q.check(Q.lib.q_b200_attn_prefix(C.byref(a), m.stream), "attn")
        torch.cuda.synchronize()
        for b in range(2):
            k = host[b, l, :, : rows[b], :32].astype(np.float64).repeat(4, 0)
            v = host[b, l, :, : rows[b], 32:].astype(np.float64).repeat(4, 0)
            y = np.einsum("hd,hld->hl", q[b].double().cpu().numpy(), k) / math.sqrt(32)
            p = np.exp(y - y.max(-1, keepdims=True))
            want = np.einsum("hl,hld->hd", p, v) / p.sum(-1, keepdims=True)
            # Y <= 32 * 4.5^2 / sqrt(32) < 128 for these draws: A (2 (2^-20 Y + 2^-21) + 2^-18) < 2^-11 A, A < 4.5
            assert np.abs(out[b].cpu().numpy() - want).max() < 4.5 * 2.0**-11
    m.close()


# ---- verification of drafts -------------------------------------------------------------------------------------------------


def do_verify(target, draft, tokens, uniform, kind="probs", temperature=1.0, length=None, dtype="f32", status=0):
    S, K1, V = target.shape
    out = torch.full((S, K1), 77, dtype=torch.int32, device="cuda")
    n = torch.full((S,), 77, dtype=torch.int32, device="cuda")
    a = Q.q_b200_verify_args(target.data_ptr(), None if draft is None else draft.data_ptr(), target.stride(0), target.stride(1),
                             0 if draft is None else draft.stride(0), 0 if draft is None else draft.stride(1),
                             tokens.data_ptr() if K1 > 1 else None, None if length is None else length.data_ptr(), uniform.data_ptr(),
                             out.data_ptr(), n.data_ptr(), S, K1 - 1, V, TYPES[dtype][1], int(kind == "logits"), temperature)
    Q.check(Q.lib.q_b200_verify_draft(C.byref(a), stream()), "q_b200_verify_draft")
    assert Q.lib.q_b200_device_status() == status
    return out.cpu().numpy(), n.cpu().numpy()


def verify64(target, draft, tokens, uniform, kind="probs", temperature=1.0, length=None):
    """The definition, one sequence after another, in 64 bits."""
    f = lambda x: None if x is None else x.double().cpu().numpy()  # noqa: E731
    target, draft, u, x = f(target), f(draft), f(uniform), tokens.cpu().numpy()
    S, K1, V = target.shape
    K, T = K1 - 1, float(np.float32(temperature))
    greedy = kind == "logits" and T < 1e-6

    def law(row):
        if kind == "probs":
            return np.where(row > 0, row, 0.0)
        ok = row[~np.isnan(row)]
        if greedy:
            return (np.arange(V) == (int(np.nanargmax(row)) if ok.size else 0)).astype(float)
        if not ok.size or ok.max() == -math.inf:
            return np.zeros(V)
        e = np.where(np.isnan(row), 0.0, np.exp((row - ok.max()) / T))
        return e / e.sum()

    out, count = np.full((S, K1), -1, np.int32), np.zeros(S, np.int32)
    for b in range(S):
        n, q = 0, None
        L = K if length is None else int(length[b])
        while n < L:
            p = law(target[b, n])
            q = law(draft[b, n]) if draft is not None and not greedy else (np.arange(V) == x[b, n]).astype(float)
            if not (x[b, n] < V and u[b, n] * q[x[b, n]] < p[x[b, n]]):
                break
            out[b, n] = x[b, n]
            n += 1
        p = law(target[b, n])
        rest = np.maximum(p - q, 0.0) if n < L and not greedy else p
        rest = rest if rest.sum() > 0 else p
        c = np.cumsum(rest)
        v = int(np.searchsorted(c, u[b, K] * c[-1], side="right"))
        out[b, n] = v if v < V else (int(np.flatnonzero(rest)[-1]) if rest.any() else 0)
        count[b] = n + 1
    return out, count


def drafted(g, S, K, V, apart=0.7, T=1.0):
    target = normal(g, S, K + 1, V) * 3
    draft = target[:, :K] + normal(g, S, K, V) * apart
    noise = torch.rand(S, K, V, generator=g, device="cuda")
    tokens = (draft / T - torch.log(-torch.log(noise))).argmax(-1).to(torch.int32) if K else torch.zeros(S, 1, dtype=torch.int32, device="cuda")
    return target, draft, tokens, torch.rand(S, K + 1, generator=g, device="cuda")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kind,T", [("probs", 1.0), ("logits", 0.7), ("logits", 0.0)])
@pytest.mark.parametrize("S,K,V", [(1, 1, 1), (3, 2, 7), (5, 4, 259), (2, 0, 1000), (17, 3, 4097), (64, 7, 2050), (1, 31, 8192), (24, 2, 50001), (2, 4, 128256),
                                   (200, 2, 515)])
def test_verify(dtype, kind, T, S, K, V):
    target, draft, tokens, u = drafted(gen(S * 100 + V), S, K, V, T=T or 1.0)
    if kind == "probs":
        target, draft = torch.softmax(target, -1), torch.softmax(draft, -1)
    target, draft = target.to(TYPES[dtype][0]), draft.to(TYPES[dtype][0])
    length = torch.randint(0, K + 1, (S,), device="cuda", dtype=torch.int32, generator=gen(1))
    for ln in (None, length):
        got, n = do_verify(target, draft if K else None, tokens, u, kind, T, ln, dtype)
        want, m = verify64(target, draft if K else None, tokens, u, kind, T, ln)
        assert np.array_equal(n, m) and np.array_equal(got, want)
    if K:  # drafts that come without probabilities
        got, n = do_verify(target, None, tokens, u, kind, T, None, dtype)
        want, m = verify64(target, None, tokens, u, kind, T, None)
        assert np.array_equal(n, m) and np.array_equal(got, want)


def test_verify_borders():
    # powers of two, so that every sum is exact: the border itself belongs to the next entry
    p = torch.tensor([[[0.25, 0.0, 0.25, 0.5]]], device="cuda")
    none = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    for u, v in ((0.0, 0), (0.2499, 0), (0.25, 2), (0.4999, 2), (0.5, 3), (0.9999, 3)):
        got, n = do_verify(p, None, none, torch.tensor([[u]], device="cuda"))
        assert n[0] == 1 and got[0, 0] == v
    # accepted while u q < p, not at u q == p
    p = torch.tensor([[[0.25, 0.75], [1.0, 0.0]]], device="cuda")
    q = torch.tensor([[[0.5, 0.5]]], device="cuda")
    x = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    assert do_verify(p, q, x, torch.tensor([[0.4999, 0.0]], device="cuda"))[0].tolist() == [[0, 0]]
    assert do_verify(p, q, x, torch.tensor([[0.5, 0.0]], device="cuda"))[0].tolist() == [[1, -1]]


def test_verify_rows_without_weight_and_not_numbers():
    nan, inf = math.nan, math.inf
    x = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    u = torch.tensor([[0.9, 0.6]], device="cuda")
    row = lambda *v: torch.tensor([[list(v)]], device="cuda")  # noqa: E731
    two = lambda a, b: torch.cat([a, b], 1)  # noqa: E731
    # p <= q everywhere and the draft refused: drawn from p itself
    assert do_verify(two(row(0.1, 0.4), row(0.5, 0.5)), row(0.5, 0.5), x, u)[0].tolist() == [[1, -1]]
    assert do_verify(two(row(0.0, 0.0), row(0.5, 0.5)), row(0.5, 0.5), x, u)[0].tolist() == [[0, -1]]
    assert do_verify(two(row(nan, 0.0, 0.3, -1.0), row(0, 0, 0, 1.0)), row(0.5, nan, 0.1, 0.0), x, u)[0].tolist() == [[2, -1]]
    # logits: masked ones at -inf, a row of nothing else, NaN
    k = dict(kind="logits", temperature=1.0)
    assert do_verify(two(row(-inf, 1.0, -inf), row(0, 0, 0)), row(0.0, -inf, -inf), x, u, **k)[0].tolist() == [[1, -1]]
    assert do_verify(two(row(-inf, -inf), row(0, 0)), row(0.0, 0.0), x, u, **k)[0].tolist() == [[0, -1]]
    assert do_verify(two(row(-inf, nan, 2.0, -inf), row(0, 0, 0, 0)), row(0.0, 0.0, -inf, 0.0), x, u, **k)[0].tolist() == [[2, -1]]
    g = dict(kind="logits", temperature=0.0)
    assert do_verify(two(row(nan, 3.0, 3.0), row(0, 0, 0)), None, x, u, **g)[0].tolist() == [[1, -1]]
    assert do_verify(two(row(3.0, 3.0, nan), row(-inf, -5.0, -5.0)), None, x, u, **g)[0].tolist() == [[0, 1]]


def test_verify_wide_temperatures():
    target, draft, tokens, u = drafted(gen(77), 4, 3, 5000)
    for T in (1e-5, 0.01, 50.0):
        got, n = do_verify(target, draft, tokens, u, "logits", T)
        want, m = verify64(target, draft, tokens, u, "logits", T)
        assert np.array_equal(n, m) and np.array_equal(got, want)


def test_verify_tokens_and_lengths_out_of_range():
    target, draft, tokens, u = drafted(gen(7), 2, 2, 50)
    target, draft = torch.softmax(target, -1), torch.softmax(draft, -1)
    tokens[0, 0] = 50
    tokens[1, 0] = -1
    got, n = do_verify(target, draft, tokens, u, status=4)
    assert n.tolist() == [1, 1] and (got[:, 0] < 50).all() and (got[:, 0] >= 0).all() and (got[:, 1:] == -1).all()
    tokens[:] = draft.argmax(-1)
    got, n = do_verify(target, draft, tokens, u, length=ints([9, 2]), status=4)
    want, m = verify64(target, draft, tokens, u)
    assert np.array_equal(got, want)


def test_verify_strided_rows_inside_a_larger_buffer():
    big = torch.softmax(normal(gen(3), 5, 9, 1003), -1)
    target, draft = big[:, 1:5, 2:902], big[:, 5:8, 3:903]
    tokens, u = draft.argmax(-1).to(torch.int32).contiguous(), torch.rand(5, 4, generator=gen(4), device="cuda")
    got, n = do_verify(target, draft, tokens, u)
    want, m = verify64(target, draft, tokens, u)
    assert np.array_equal(n, m) and np.array_equal(got, want)


# ---- together -------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_speculative_step(dtype):
    """Drafted tokens of three sequences behind a shared prompt: rotated and appended, attended, projected to logits, verified;
    then the accepted rows' lengths are what the next step starts from.  One captured graph, two steps."""
    H, KV, D, R, P, V, K = 8, 2, 64, 16, 100, 300, 3
    b = Batch(31, dtype, H, KV, D, R, P, [30, 17, 64], [K + 1] * 3, room_rows=40, poison=False)
    g, p = gen(32), make_plan(D, "half", "banded")
    t = torch.arange(3 * (K + 1), device="cuda")
    seq = (t // (K + 1)).to(torch.int32)
    head = normal(g, H * D, V) * 0.2
    state = dict(lens=[30, 17, 64])
    qkv = torch.zeros(3 * (K + 1), H + 2 * KV, D, dtype=TYPES[dtype][0], device="cuda")
    q, k, v = qkv[:, :H], qkv[:, H: H + KV], qkv[:, H + KV:]
    q_rot, row, pos = torch.empty_like(q), ints([0] * len(t)), ints([0] * len(t))
    b.q = q_rot
    logits = torch.empty(3, K + 1, V, device="cuda")
    draft, drafts, u = torch.empty(3, K, V, device="cuda"), ints([[0] * K] * 3), torch.empty(3, K + 1, device="cuda")
    chosen, count = ints([[0] * (K + 1)] * 3), ints([0] * 3)
    attn = b.args(max_len=104)
    ver = Q.q_b200_verify_args(logits.data_ptr(), draft.data_ptr(), logits.stride(0), V, draft.stride(0), V, drafts.data_ptr(), None,
                               u.data_ptr(), chosen.data_ptr(), count.data_ptr(), 3, K, V, Q.Q_B200_F32, Q.Q_B200_LOGITS, 0.9)

    def step():
        do_append(b.keys, b.values, dtype, k, v, b.pages, seq, row, pos, p, dtype, q, q_rot)
        Q.check(Q.lib.q_b200_attn_prefix(C.byref(attn), stream()), "attn")
        logits.copy_(torch.matmul(b.out.float().view(-1, H * D), head).view(3, K + 1, V))
        Q.check(Q.lib.q_b200_verify_draft(C.byref(ver), stream()), "verify")

    step()  # libraries settle before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for n in range(2):
        qkv.copy_(normal(g, *qkv.shape, dtype=dtype))
        draft.copy_(normal(g, 3, K, V))
        drafts.copy_(torch.randint(0, V, (3, K), generator=g, device="cuda"))
        u.copy_(torch.rand(3, K + 1, generator=g, device="cuda") * 0.2)
        at = torch.tensor(state["lens"], device="cuda")[seq.long()] + t % (K + 1)
        row.copy_(at)
        pos.copy_(at + P)
        b.rows = [x + K + 1 for x in state["lens"]]
        b.lens.copy_(ints(b.rows))
        pool = b.pool.clone()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        # each operator against 64 bits on what it was given
        want, room = turn64(q, pos, p)
        within(q_rot, want, room, dtype)
        page = b.pages[seq.long(), at // R].long()
        want, room = turn64(k, pos, p)
        within(b.keys.permute(0, 2, 1, 3)[page, at % R], want, room, dtype)
        assert not torch.equal(pool, b.pool)
        want, room = b.want()
        within(b.out, want, room, dtype)
        got, m = verify64(logits, draft, drafts, u, "logits", 0.9)
        assert np.array_equal(chosen.cpu().numpy(), got) and np.array_equal(count.cpu().numpy(), m)
        state["lens"] = [x + int(c) for x, c in zip(state["lens"], count.cpu())]
    assert Q.lib.q_b200_device_status() == 0


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_steps_without_a_wait_between_them(dtype):
    """Each call reads what the one before it has written, twenty steps behind one another: the same bits as with a wait after
    every call (the kernels may be set up beside the tail of the work before them)."""
    H, KV, D, B, V = 16, 2, 64, 3, 500
    g, p = gen(50), make_plan(D, "half")
    b = Batch(51, dtype, H, KV, D, 16, 200, [1] * B, [1] * B, room_rows=40, poison=False)
    pool = b.pool.clone()
    xs = normal(g, 20, B, H + 2 * KV, D, dtype=dtype)
    head = normal(g, H * D, V) * 0.3
    u = torch.rand(B, 1, generator=g, device="cuda")
    q, turned = torch.empty_like(xs[0][:, :H]), torch.empty_like(xs[0][:, :H])
    b.q = turned
    a = b.args(max_len=40)

    def run(wait):
        b.pool.copy_(pool)
        b.lens.fill_(1)
        row, seen = ints([0] * B), []
        torch.cuda.synchronize()
        for x in xs:
            q.copy_(x[:, :H])
            do_append(b.keys, b.values, dtype, x[:, H:H + KV], x[:, H + KV:], b.pages, None, row, None, p, dtype)
            if wait: torch.cuda.synchronize()
            do_rope(q, turned, row, p, dtype=dtype)
            do_rope(turned, turned, row, p, dtype=dtype)
            if wait: torch.cuda.synchronize()
            Q.check(Q.lib.q_b200_attn_prefix(C.byref(a), stream()), "attn")
            Q.check(Q.lib.q_b200_attn_prefix(C.byref(a), stream()), "attn")
            if wait: torch.cuda.synchronize()
            logits = torch.matmul(b.out.float().view(B, H * D), head).view(B, 1, V)
            out, n = ints([[0]] * B), ints([0] * B)
            v = Q.q_b200_verify_args(logits.data_ptr(), None, V, V, 0, 0, None, None, u.data_ptr(), out.data_ptr(), n.data_ptr(), B, 0, V,
                                     0, Q.Q_B200_LOGITS, 1.0)
            Q.check(Q.lib.q_b200_verify_draft(C.byref(v), stream()), "verify")
            seen += [b.out.clone(), out.clone()]
            if wait: torch.cuda.synchronize()
            row += 1
            b.lens += 1
        torch.cuda.synchronize()
        return seen + [b.pool.clone()]

    slow, fast = run(True), run(False)
    assert all(torch.equal(x, y) for x, y in zip(slow, fast))
    assert Q.lib.q_b200_device_status() == 0


def test_calls_on_two_streams_at_once():
    streams, jobs = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(2):
        g = gen(60 + i)
        x, p = normal(g, 3000, 8, 128, dtype="bf16"), make_plan(128)
        pos = torch.randint(0, 5000, (3000,), generator=g, device="cuda", dtype=torch.int32)
        target, draft, tokens, u = drafted(g, 20, 3, 20000)
        jobs.append((x, torch.empty_like(x), pos, p, target, draft, tokens, u, torch.zeros(20, 4, dtype=torch.int32, device="cuda"),
                     torch.zeros(20, dtype=torch.int32, device="cuda")))
    torch.cuda.synchronize()
    for _ in range(5):
        for s, (x, out, pos, p, target, draft, tokens, u, chosen, n) in zip(streams, jobs):
            do_rope(x, out, pos, p, dtype="bf16", on=s.cuda_stream)
            v = Q.q_b200_verify_args(target.data_ptr(), draft.data_ptr(), 4 * 20000, 20000, 3 * 20000, 20000, tokens.data_ptr(), None, u.data_ptr(),
                                     chosen.data_ptr(), n.data_ptr(), 20, 3, 20000, 0, Q.Q_B200_LOGITS, 0.8)
            Q.check(Q.lib.q_b200_verify_draft(C.byref(v), s.cuda_stream), "verify")
    torch.cuda.synchronize()
    for x, out, pos, p, target, draft, tokens, u, chosen, n in jobs:
        want, room = turn64(x, pos, p)
        within(out, want, room, "bf16")
        got, m = verify64(target, draft, tokens, u, "logits", 0.8)
        assert np.array_equal(chosen.cpu().numpy(), got) and np.array_equal(n.cpu().numpy(), m)


@pytest.mark.parametrize("call", ["rope", "append", "attn", "verify"])
def test_host_memory_is_refused(call):
    x = torch.zeros(4, 2, 64)
    d = x.cuda()
    i, p = ints([0, 0, 0, 0]), make_plan(64)
    if call == "rope":
        a = Q.q_b200_rope_args(x.data_ptr(), d.data_ptr(), i.data_ptr(), C.addressof(p), 128, 64, 128, 64, 4, 2, 64, 0, 0, 0)
        assert Q.lib.q_b200_rope(C.byref(a), None) == -10
    elif call == "append":
        with pytest.raises(Q.QorusError, match="INVALID_ARG"):
            do_append(d.view(4, 2, 1, 64), d.view(4, 2, 1, 64), "f32", d, x, i.view(4, 1), None, i, None, p, "f32")
    elif call == "attn":
        b = Batch(1, "f32", 2, 1, 64, 16, 0, [3], [1])
        b.lens = b.lens.cpu()
        with pytest.raises(Q.QorusError, match="INVALID_ARG"):
            b.call()
    else:
        with pytest.raises(Q.QorusError, match="INVALID_ARG"):
            do_verify(d, None, i[:4].view(4, 1).cpu().repeat(1, 1), torch.zeros(4, 2, device="cuda"))
    assert "current device" in Q.last_error()
