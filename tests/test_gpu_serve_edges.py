"""The serving operators at values, lengths and tables past those of test_gpu_serve.py, whose helpers and tolerances they use."""
import ctypes as C
import math

import numpy as np
import pytest

import qorus_b200 as Q

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_gpu_serve import TYPES, Batch, do_verify, gen, half_step, ints, make_plan, turn64, verify64, within  # noqa: E402

# ---- attention -------------------------------------------------------------------------------------------------------


def weighted(b):
    """(result, room) of one token a sequence, as Batch.want gives them, with scores of -infinity: a row of weight zero adds
    nothing, whatever its value, and a vector without any weight gives zeros."""
    G, outs, rooms = b.heads // b.keys.shape[1], [], []
    flat = lambda x, p: x[p.long()].transpose(1, 2).reshape(-1, x.shape[1], b.dim).double()  # noqa: E731
    for i, L in enumerate(b.rows):
        k, v = (torch.cat([flat(x, b.prefix_pages)[: b.prefix], flat(x, b.pages[i])[:L]]).repeat_interleave(G, 1) for x in (b.keys, b.values))
        q = b.q[i].double()
        y = torch.einsum("hd,lhd->hl", q, k) / math.sqrt(b.dim)
        p = torch.softmax(y, -1).nan_to_num(0.0)
        v = torch.where(p.T[..., None] > 0, v, 0.0)
        o, A = torch.einsum("hl,lhd->hd", p, v), torch.einsum("hl,lhd->hd", p, v.abs())
        size = torch.einsum("hd,lhd->hl", q.abs(), k.abs()) / math.sqrt(b.dim)
        Y = torch.where(p > 0, size, 0.0).amax(-1, keepdim=True)
        room = A * (2 * (2.0**-20 * Y + 2.0**-21) + 2.0**-18)
        outs.append(o)
        rooms.append(room if b.dtype == "f32" else room + half_step(b.dtype) * (A + o.abs()))
    return torch.stack(outs), torch.stack(rooms)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim,prefix,seqs", [
    (8, 2, 64, 200, 3), (24, 2, 128, 200, 2),                        # up to 16 and 32 vectors of a KV head,
    (32, 2, 64, 300, 5), (64, 2, 128, 300, 9), (64, 2, 64, 300, 9),  # up to 128 and more
    (64, 2, 32, 130, 4), (8, 2, 128, 0, 3)])                         # without tcgen05, without a prefix
def test_attn_scores_of_minus_infinity(dtype, heads, kv_heads, dim, prefix, seqs):
    top = torch.finfo(TYPES[dtype][0]).max
    b = Batch(dim + seqs, dtype, heads, kv_heads, dim, 16, prefix, [20 + i for i in range(seqs)], [1] * seqs, poison=False)
    b.q[..., 0] = b.q[..., 0].abs() + 0.5  # a key of -infinity scores -infinity
    keys, values = b.keys.clone(), b.values.clone()
    off = torch.rand(b.keys.shape[0], kv_heads, 16, generator=gen(1), device="cuda")
    for part, huge in ((0.3, True), (0.9, True), (2.0, False)):  # some rows, most of them, every row
        for h in (0, 1):  # every row of the first KV head's, some of the second's
            gone = off[:, h] < (part if h == 0 else part / 3)
            b.keys[:, h, :, 0] = torch.where(gone, -math.inf, keys[:, h, :, 0])
            if huge:
                b.values[:, h] = torch.where(gone[..., None], top, values[:, h])
            else:
                b.values[:, h] = values[:, h]
        b.call()
        want, room = weighted(b)
        if not huge:
            assert (want[:, : heads // kv_heads] == 0).all()
        within(b.out, want, room, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads", [8, 40])
@pytest.mark.parametrize("sign", [-1, 1])
def test_attn_newer_rows_of_the_types_largest_numbers_do_not_reach_older_tokens(dtype, heads, sign):
    b = Batch(4, dtype, heads, 2, 64, 16, 100, [90, 8], [6, 5], poison=False)
    b.call()
    clean = b.out.clone()
    for x in (b.keys, b.values):
        for r in (88, 89):
            x[b.pages[0, r // 16].long(), :, r % 16] = sign * torch.finfo(x.dtype).max
        x[b.pages[1, 0].long(), :, 7] = sign * torch.finfo(x.dtype).max
    b.call()
    assert torch.equal(b.out[:4], clean[:4]) and torch.equal(b.out[6:10], clean[6:10])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads", [8, 80])
def test_attn_one_row_of_the_types_largest_numbers(dtype, heads):
    # alone it is the result itself; beside keys that score more it weighs nothing
    b = Batch(5, dtype, heads, 2, 64, 16, 0, [1, 40], [1, 1], poison=False)
    top = torch.finfo(TYPES[dtype][0]).max
    b.q[..., 0] = b.q[..., 0].abs() + 0.5
    for i in range(2):
        page = b.pages[i, 0].long()
        b.values[page, :, 0] = torch.where(torch.arange(64, device="cuda") % 2 == 0, top, -top).to(b.values.dtype)
        b.keys[page, :, 0, 0] = -top / 64  # q.k is finite
    b.call()
    # fp32's largest number has 24 bits, of which its two halves hold 11 each: off by 2^-22, within the room for products
    want, room = weighted(b)
    assert want[0].abs().min() == top
    within(b.out, want, room, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,seqs,rows,prefix", [
    (400, 100, 4, 1 << 20, 0), (320, 8, 4, 1 << 20, 0), (4, 1, 1, 300000, 0),         # own rows: up to 32 vectors, more, one sequence
    (1280, 160, 9, 300, 1 << 20), (1280, 160, 40, 300, 1 << 18), (320, 160, 3, 20, 1 << 20)])  # the prefix: up to 128 vectors, more, few
def test_attn_sums_of_many_rows(dtype, heads, kv_heads, seqs, rows, prefix):
    # A page table that names the same pages again and again.  Queries of zero weigh all rows alike, exactly, so the result is the
    # values' own: off by what the sums lose (a product truncates its sum by two steps of 2^-24 of it at most, half of that on the
    # average over a growing sum, 512 of them, or 1024 that truncate once; fp32 rounds 1024 times by 2^-24 at most) and by one rounding.
    b = Batch(2, dtype, heads, kv_heads, 64, 16, 288, [288] * seqs, [1] * seqs, poison=False)
    b.q = torch.zeros_like(b.q)
    value = torch.linspace(0.3, 3.0, 64, device="cuda").to(TYPES[dtype][0])
    b.values.copy_(value.expand_as(b.values))
    again = lambda p, n: p[..., torch.arange(-(-n // 16), device="cuda") % 18].contiguous()  # noqa: E731
    b.pages, b.prefix_pages = again(b.pages, rows), again(b.prefix_pages, prefix) if prefix else b.prefix_pages
    b.per, b.rows, b.prefix = b.pages.shape[1], [rows - i for i in range(seqs)], prefix
    b.lens, b.prefix_len = ints(b.rows), ints([prefix])
    b.call()
    want = value.double().expand(seqs, heads, 64)
    within(b.out, want, want * 2.0**-14, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim,prefix,seqs", [
    (8, 2, 64, 8000, 3), (24, 2, 128, 8000, 2), (32, 2, 64, 8000, 5), (64, 2, 128, 8000, 9), (64, 2, 32, 8000, 4), (8, 2, 128, 0, 3), (80, 2, 64, 0, 2),
    (320, 160, 64, 4000, 3)])  # so many KV heads that a warp takes a quarter of all rows
@pytest.mark.parametrize("sink", [0, -1])
def test_attn_weights_far_below_the_largest(dtype, heads, kv_heads, dim, prefix, seqs, sink):
    # one row that outweighs each of the thousands of others by 2^14 to 2^28, and has no value of its own, as the first token of a
    # prompt often does: the others are the result.  16 bits lose nothing but their own step of fp16 weights (2^-25, where the
    # largest is 2^7 at least): 2^-32 of it for each row.
    rows = 8000 if not prefix else 20
    b = Batch(dim + seqs, dtype, heads, kv_heads, dim, 16, prefix, [rows] * seqs, [1] * seqs, poison=False)
    b.q.zero_()
    b.q[..., 0] = 1.0
    b.keys[..., 0] *= 0.25
    b.values.add_(1.0)
    pages = [b.prefix_pages] if prefix else list(b.pages)
    n = prefix or rows
    at = 0 if sink == 0 else n - 1
    for gap in (14.0, 18.3, 22.5, 25.4, 28.0):
        for p in pages:
            b.keys[p[at // 16].long(), :, at % 16, 0] = gap * math.log(2) * math.sqrt(dim)
            b.values[p[at // 16].long(), :, at % 16] = 0.0
        b.call()
        want, room = weighted(b)
        within(b.out, want, room + (2.0**-32 * (prefix + rows) * float(b.values.abs().max()) if dtype == "f16" else 0.0), dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim,seqs", [(8, 2, 64, 3), (24, 2, 128, 2), (32, 2, 64, 5), (64, 2, 128, 9), (64, 2, 32, 4)])
def test_attn_largest_values_behind_smaller_scores(dtype, heads, kv_heads, dim, seqs):
    # the last row of the prefix weighs 2^7.5 times each other and has the type's largest values: its share of them is finite
    b = Batch(dim + seqs, dtype, heads, kv_heads, dim, 16, 200, [20] * seqs, [1] * seqs, poison=False)
    b.q.zero_()
    b.q[..., 0] = 1.0
    b.keys[..., 0] = 0.0
    page = b.prefix_pages[199 // 16].long()
    b.keys[page, :, 199 % 16, 0] = 7.5 * math.log(2) * math.sqrt(dim)
    b.values[page, :, 199 % 16] = torch.finfo(TYPES[dtype][0]).max
    b.call()
    want, room = weighted(b)
    assert torch.isfinite(want).all()
    within(b.out, want, room, dtype)


@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f16", 64)])
@pytest.mark.parametrize("G,seqs,prefix", [(4, 20, 4100), (4, 40, 4173), (1, 300, 6143), (2, 64, 12289)])
def test_attn_prefix_parts_of_many_tiles(dtype, dim, G, seqs, prefix):
    # 160 KV heads leave one part each: 33 tiles of 128 rows and more in one CTA, so that its ring of 5 or 9 slots and all of its
    # barriers go round many times, for one tile of vectors (80, 128) and two (160, 300)
    KV, L, R = 160, 3, 32
    g = gen(prefix)
    shared = -(-prefix // R)
    pool = torch.randn(shared + seqs, KV, R, 2 * dim, generator=g, device="cuda", dtype=torch.float16).to(TYPES[dtype][0])
    keys, values = pool[..., :dim], pool[..., dim:]
    q = torch.randn(seqs, KV * G, dim, generator=g, device="cuda").to(TYPES[dtype][0])
    out, ids = torch.zeros_like(q), torch.randperm(shared + seqs, generator=g, device="cuda").to(torch.int32)
    prefix_pages, pages, lens, n = ids[:shared].contiguous(), ids[shared:].contiguous(), ints([L] * seqs), ints([prefix])
    kv = Q.q_b200_paged_kv(keys.data_ptr(), values.data_ptr(), pool.stride(0), pool.stride(1), pool.stride(2), shared + seqs, R, KV, dim,
                           TYPES[dtype][1], 0)
    a = Q.q_b200_attn_args(kv, q.data_ptr(), out.data_ptr(), q.stride(0), dim, q.stride(0), dim, None, pages.data_ptr(), lens.data_ptr(),
                           prefix_pages.data_ptr(), n.data_ptr(), None, 0, seqs, seqs, KV * G, 1, 1, L, prefix, 1 / math.sqrt(dim))
    work = torch.empty(Q.lib.q_b200_attn_work_bytes(C.byref(a)), dtype=torch.uint8, device="cuda")
    assert work.numel() == seqs * KV * G * (dim * 4 + 8)  # one part
    a.work, a.work_bytes = work.data_ptr(), work.numel()
    Q.check(Q.lib.q_b200_attn_prefix(C.byref(a), torch.cuda.current_stream().cuda_stream), "attn")
    assert Q.lib.q_b200_device_status() == 0
    for h in range(0, KV, 9):
        rows = lambda x: torch.cat([x[prefix_pages.long(), h].reshape(-1, dim)[:prefix].expand(seqs, -1, -1), x[pages.long(), h, :L]], 1)  # noqa: E731
        k, v, x = rows(keys).double(), rows(values).double(), q[:, h * G: (h + 1) * G].double()
        y = x @ k.transpose(1, 2) / math.sqrt(dim)
        w = torch.softmax(y, -1)
        o, A = w @ v, w @ v.abs()
        Y = (x.abs() @ k.abs().transpose(1, 2) / math.sqrt(dim)).amax(-1, keepdim=True)
        # the rooms of test_gpu_serve.py with what this pass adds: a quarter of the exponentials good to 5.6e-5 < 2^-14, and a sum
        # that up to 1024 products truncate, by 2^-24 of it each on the average
        room = A * (2 * (2.0**-20 * Y + 2.0**-14) + 2.0**-14) + half_step(dtype) * (A + o.abs())
        within(out[:, h * G: (h + 1) * G], o, room, dtype)


# ---- the batch's own pages ---------------------------------------------------------------------------------------------


def test_rows_appended_through_the_view_are_the_frameworks_own(tmp_path):
    cfg = Q.config(vocab=259, dim=256, hidden=512, layers=2, heads=8, kv_heads=2, max_seq=256)
    Q.write_model(str(tmp_path / "m.qorus"), cfg, seed=0, threads=1)
    N, hd = 130, 32
    ms = [Q.Model(str(tmp_path / "m.qorus")) for _ in range(2)]
    for m in ms:
        Q.check(Q.lib.q_b200_batch_init_paged(C.byref(m.ctx), C.byref(m.model), 2, 128, 6), "batch_init_paged")
    first, second = ms
    vocab, logits, nxt = cfg.vocab_size, [np.zeros((2, cfg.vocab_size), np.float32) for _ in ms], [np.zeros(2, np.uint32) for _ in ms]

    def decode(i, tokens, pos):
        t, p = np.array(tokens, np.uint32), np.array(pos, np.uint32)
        Q.check(Q.lib.q_b200_decode_batch(C.byref(ms[i].model), C.byref(ms[i].ctx), Q.ptr(t), Q.ptr(p), Q.ptr(logits[i]), Q.ptr(nxt[i])), "decode")

    rng = np.random.default_rng(0)
    tokens = rng.integers(0, vocab, (N, 2))
    tokens[100] = tokens[0]  # the same tokens at row 0, where nothing turns, and at row 100
    for n in range(N):
        decode(0, tokens[n], [n, n])
    rows = np.zeros((2, 2, 2, 256, 2 * hd), np.float32)  # [seq][layer][head][row][K|V]
    for b in range(2):
        Q.check(Q.lib.q_b200_batch_kv_read(C.byref(first.ctx), b, 0, Q.ptr(rows[b]), rows[b].nbytes), "kv_read")
    none = np.zeros((N, 2 * hd), np.float32)
    for b in range(2):  # rows that are written take pages
        Q.check(Q.lib.q_b200_batch_kv_write(C.byref(second.ctx), b, 0, Q.ptr(none), none.nbytes), "kv_write")
    kv, pages, per = Q.q_b200_paged_kv(), C.c_void_p(), C.c_uint32()
    seq, row = ints([b for b in range(2) for _ in range(N)]), ints(list(range(N)) * 2)

    def append(layer, k, v, seq, row, plan):
        Q.check(Q.lib.q_b200_batch_kv_view(C.byref(second.ctx), layer, C.byref(kv), C.byref(pages), C.byref(per)), "view")
        a = Q.q_b200_append_args(kv, k.data_ptr(), v.data_ptr(), None, None, k.stride(0), k.stride(1), v.stride(0), v.stride(1), 0, 0, 0, 0, pages,
                                 seq.data_ptr(), row.data_ptr(), None, C.addressof(plan) if plan else None, len(row), 2, per.value, 0, Q.Q_B200_F32, 0)
        torch.cuda.synchronize()
        Q.check(Q.lib.q_b200_kv_append(C.byref(a), second.stream), "append")
        torch.cuda.synchronize()

    # rotation: the framework's row 0 (layer 0 knows the token alone), turned to row 100 here, is the framework's row 100.  Its angles
    # are fp32 products: off by 100 * 2^-22 (frequency and product), beside what turn64 allows for this side
    plan = make_plan(hd, "interleaved")
    raw = torch.from_numpy(rows[:, 0, :, 0]).cuda()
    append(0, raw[..., :hd], raw[..., hd:], ints([0, 1]), ints([100, 100]), plan)
    mine = np.zeros((2, 256, 2 * hd), np.float32)
    for b in range(2):
        Q.check(Q.lib.q_b200_batch_kv_read(C.byref(second.ctx), b, 0, Q.ptr(mine), mine.nbytes), "kv_read")
        want, room = turn64(raw[b:b + 1, :, :hd], ints([100]), plan)
        got = torch.from_numpy(mine[:, 100]).cuda()
        within(got[None, :, :hd], want, room, "f32")
        theirs = torch.from_numpy(rows[b, 0, :, 100]).cuda().double()
        assert ((got[:, :hd].double() - theirs[:, :hd]).abs() <= 2 * room[0] * (1 + 100 * 2.0**-22 / 2.0**-20)).all()
        assert torch.equal(got[:, hd:].double(), theirs[:, hd:])
    # the framework's rows, appended as they are: the next step has the same bits
    for layer in range(2):
        x = torch.from_numpy(rows[:, layer, :, :N]).cuda().transpose(1, 2).reshape(2 * N, 2, 2 * hd)
        append(layer, x[..., :hd], x[..., hd:], seq, row, None)
    for step in range(3):
        for i in range(2):
            decode(i, nxt[i] if step else tokens[0], [N + step] * 2)
        assert np.array_equal(logits[0], logits[1]) and np.array_equal(nxt[0], nxt[1])
    # a row past the pages that the sequence has is skipped: the view takes none
    assert Q.lib.q_b200_device_status() == 0
    x = torch.ones(1, 2, 2 * hd, device="cuda")
    append(0, x[..., :hd], x[..., hd:], ints([1]), ints([256]), None)
    assert Q.lib.q_b200_device_status() == 4
    Q.check(Q.lib.q_b200_batch_release(C.byref(second.ctx), 1), "release")
    append(0, x[..., :hd], x[..., hd:], ints([1]), ints([0]), None)
    assert Q.lib.q_b200_device_status() == 4
    for m in ms:
        m.close()


# ---- verification of drafts ------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V,first,second", [(3, 0, 1), (259, 17, 18), (8192, 40, 4099), (128256, 5, 100003)])
def test_verify_greedy_takes_the_first_of_two_zeros(dtype, V, first, second):
    # -0 and +0 are equal: whichever sign comes first, the first of them is the first maximum
    u = torch.full((1, 2), 0.5, device="cuda")
    for a, b in ((-0.0, 0.0), (0.0, -0.0), (-0.0, -0.0)):
        target = torch.full((1, 2, V), -1.0, device="cuda")
        target[..., first], target[..., second] = a, b
        for drafted, want in ((first, [first, first]), (second, [first, -1])):
            got, n = do_verify(target.to(TYPES[dtype][0]), None, ints([[drafted]]), u, "logits", 0.0, None, dtype)
            assert got.tolist() == [want] and n[0] == 1 + (drafted == first)


@pytest.mark.parametrize("T", [1e-6, 1e-5, 0.8, 3.0])
@pytest.mark.parametrize("dtype,offset,spread", [
    # a step of fp32 is more than a thousand halvings at the lowest temperatures
    *((d, 2e4, 3.0) for d in ("f32", "f16", "bf16")), *((d, 6e4, 3000.0) for d in ("f32", "f16", "bf16")),
    *((d, x, y) for d in ("f32", "bf16") for x, y in ((-3e5, 3.0), (-1e9, 1e3))),
    # all alike, as in a row that is masked as a whole: uniform
    ("f32", 1e30, 0.0), ("bf16", 1e30, 0.0), *((d, x, 0.0) for d in ("f32", "f16", "bf16") for x in ("lowest", "largest"))])
def test_verify_logits_far_from_zero(dtype, T, offset, spread):
    V, top = 1000, torch.finfo(TYPES[dtype][0]).max
    base = {"lowest": -top, "largest": top}.get(offset, offset)
    target = base + spread * torch.rand(1, 2, V, generator=gen(1), device="cuda", dtype=torch.float64)
    target = target.to(TYPES[dtype][0])
    target[0, :, 7], target[0, :, 8] = -float("inf"), float("nan")
    x, u = ints([[3]]), torch.tensor([[0.9, 0.6004]], device="cuda")  # 0.6004 of 997 or 998 equal weights is inside an entry
    for t, draft, xs, us in ((target, None, x, u), (target[:, :1].contiguous(), None, x, u[:, 1:].contiguous()),
                             (target, target[:, 1:].roll(1, -1).contiguous(), x, u)):
        if spread == 0 and draft is not None:
            continue  # p - q of equal rows is a matter of rounding
        got, n = do_verify(t, draft, xs, us, "logits", T, None, dtype)
        # the record's 1e-6 is the fp32 number, which is not below itself: the oracle, which compares it in 64 bits, gets the next one
        # (weights of so low a temperature are one or zero with either)
        want, m = verify64(t, draft, xs, us, "logits", float(np.nextafter(np.float32(T), np.float32(1))) if T == 1e-6 else T)
        assert np.array_equal(n, m) and np.array_equal(got, want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("S,K,V", [(1, 0, 5000), (1, 2, 128256), (40, 1, 20001)])
def test_verify_weights_whose_sum_passes_fp32(dtype, S, K, V):
    # rows of weights need not sum to one, nor to anything that fp32 holds
    g = gen(V)
    target = (torch.rand(S, K + 1, V, generator=g, device="cuda") * 3e38).to(TYPES[dtype][0])
    draft = (torch.rand(S, K, V, generator=g, device="cuda") * 3e38).to(TYPES[dtype][0]) if K else None
    x = torch.randint(0, V, (S, max(1, K)), generator=g, device="cuda", dtype=torch.int32)
    u = torch.rand(S, K + 1, generator=g, device="cuda")
    for d in (draft, None):
        got, n = do_verify(target, d, x, u, "probs", 1.0, None, dtype)
        want, m = verify64(target, d, x, u)
        assert np.array_equal(n, m) and np.array_equal(got, want)
