"""The serving operators' argument checks and frequency plans, without a GPU: no call here launches a kernel.

The pointers are numbers that nothing looks behind: each refusal comes before the device is asked, and a record
that passes every check is refused last because its pointers are no device's."""
import ctypes as C
import math

import numpy as np
import pytest

import qorus_b200 as Q

OK, ARG, ALIAS, ALIGN, DTYPE, SIZE = 0, -10, -11, -13, -14, -15
P = 1 << 20  # an aligned address that is no memory


def cache(**kw):
    c = dict(k=P, v=P + 512, page_stride=16384, head_stride=8192, row_stride=256, n_pages=4, page_rows=32, n_kv_heads=2,
             head_dim=128, dtype=Q.Q_B200_F32, reserved=0)
    c.update(kw)
    return Q.q_b200_paged_kv(**c)


def plan(rot=128, layout=Q.Q_B200_ROPE_HALF, base=10000.0, scale=None):
    p = Q.q_b200_rope_plan()
    assert Q.lib.q_b200_rope_plan_init(C.byref(p), rot, layout, base, scale and C.byref(scale)) == OK
    return p


PLAN = plan()


def rope(**kw):
    a = dict(x=P, out=2 * P, pos=3 * P, plan=C.addressof(PLAN), x_token_stride=256, x_head_stride=128, out_token_stride=256,
             out_head_stride=128, n_tokens=3, n_heads=2, head_dim=128, dtype=Q.Q_B200_F32, transpose=0, reserved=0)
    a.update(kw)
    return Q.lib.q_b200_rope(C.byref(Q.q_b200_rope_args(**a)), None)


def append(**kw):
    a = dict(kv=cache(), k=P, v=2 * P, q=None, q_out=None, k_token_stride=256, k_head_stride=128, v_token_stride=256,
             v_head_stride=128, q_token_stride=512, q_head_stride=128, q_out_token_stride=512, q_out_head_stride=128,
             pages=3 * P, seq=4 * P, row=5 * P, pos=None, plan=C.addressof(PLAN), n_tokens=3, n_seqs=2, pages_per_seq=2,
             n_heads=4, dtype=Q.Q_B200_F32, reserved=0)
    a.update(kw)
    return Q.lib.q_b200_kv_append(C.byref(Q.q_b200_append_args(**a)), None)


def attn_args(**kw):
    a = dict(kv=cache(), q=P, out=2 * P, q_token_stride=512, q_head_stride=128, out_token_stride=512, out_head_stride=128,
             q_start=None, pages=3 * P, lens=4 * P, prefix_pages=5 * P, prefix_len=6 * P, work=7 * P, work_bytes=1 << 40,
             n_tokens=2, n_seqs=2, n_heads=4, pages_per_seq=2, max_q=1, max_len=64, max_prefix=128, scale=0.1)
    a.update(kw)
    return Q.q_b200_attn_args(**a)


def attn(**kw):
    return Q.lib.q_b200_attn_prefix(C.byref(attn_args(**kw)), None)


def verify(**kw):
    a = dict(target=P, draft=2 * P, target_seq_stride=5000, target_row_stride=1000, draft_seq_stride=4000,
             draft_row_stride=1000, draft_tokens=3 * P, draft_len=None, uniform=4 * P, tokens=5 * P, n_tokens=6 * P, n_seqs=2,
             n_draft=4, vocab=1000, dtype=Q.Q_B200_F32, kind=Q.Q_B200_PROBS, temperature=1.0)
    a.update(kw)
    return Q.lib.q_b200_verify_draft(C.byref(Q.q_b200_verify_args(**a)), None)


def test_null_records():
    for f in (Q.lib.q_b200_rope, Q.lib.q_b200_kv_append, Q.lib.q_b200_attn_prefix, Q.lib.q_b200_verify_draft):
        assert f(None, None) == ARG
    assert Q.lib.q_b200_attn_work_bytes(None) == 0


@pytest.mark.parametrize("call", [rope, append, attn, verify])
def test_pointers_that_are_no_device_memory(call):
    assert call() == ARG


@pytest.mark.parametrize("kw,rc", [
    (dict(x=None), ARG), (dict(out=None), ARG), (dict(pos=None), ARG), (dict(plan=None), ARG), (dict(dtype=3), DTYPE),
    (dict(reserved=1), ARG), (dict(transpose=2), ARG), (dict(n_tokens=0), SIZE), (dict(n_heads=0), SIZE), (dict(head_dim=0), SIZE),
    (dict(head_dim=257), SIZE), (dict(head_dim=64), SIZE), (dict(n_heads=65536), SIZE), (dict(x_token_stride=1 << 32), SIZE), (dict(x=P + 2), ALIGN), (dict(out=P + 1, dtype=1), ALIGN),
    (dict(pos=P + 2), ALIGN), (dict(out=P, out_head_stride=256), ALIAS)])
def test_rope_refuses(kw, rc):
    assert rope(**kw) == rc


@pytest.mark.parametrize("kw,rc", [
    (dict(k=None), ARG), (dict(v=None), ARG), (dict(pages=None), ARG), (dict(row=None), ARG), (dict(kv=cache(k=None)), ARG),
    (dict(kv=cache(dtype=7)), DTYPE), (dict(kv=cache(reserved=1)), ARG), (dict(kv=cache(n_pages=0)), SIZE),
    (dict(kv=cache(page_rows=0)), SIZE), (dict(kv=cache(n_kv_heads=0)), SIZE), (dict(kv=cache(row_stride=64)), SIZE),
    (dict(kv=cache(v=P + 2)), ALIGN), (dict(kv=cache(head_dim=512, row_stride=512)), SIZE), (dict(dtype=5), DTYPE),
    (dict(n_tokens=0), SIZE), (dict(n_seqs=0), SIZE), (dict(pages_per_seq=0), SIZE), (dict(seq=None), SIZE),
    (dict(q=P, q_out=None), ARG), (dict(q=P, q_out=2 * P, n_heads=0), SIZE), (dict(q=P, q_out=P, q_out_head_stride=64), ALIAS),
    (dict(kv=cache(head_dim=64)), SIZE), (dict(row=P + 1), ALIGN), (dict(reserved=9), ARG),
    (dict(kv=cache(head_stride=1 << 32)), SIZE), (dict(v_token_stride=1 << 40), SIZE), (dict(q=P, q_out=2 * P, n_heads=70000), SIZE)])
def test_append_refuses(kw, rc):
    assert append(**kw) == rc


@pytest.mark.parametrize("kw,rc", [
    (dict(q=None), ARG), (dict(out=None), ARG), (dict(pages=None), ARG), (dict(lens=None), ARG), (dict(prefix_pages=None), ARG),
    (dict(prefix_len=None), ARG), (dict(kv=cache(head_dim=96)), SIZE), (dict(kv=cache(dtype=4)), DTYPE),
    (dict(kv=cache(row_stride=130)), ALIGN), (dict(kv=cache(page_rows=0)), SIZE), (dict(n_heads=5), SIZE), (dict(n_heads=0), SIZE),
    (dict(n_tokens=0), SIZE), (dict(n_seqs=0), SIZE), (dict(max_q=0), SIZE), (dict(n_tokens=3), SIZE), (dict(max_q=2), SIZE),
    (dict(max_len=65), SIZE), (dict(max_prefix=1 << 30), SIZE), (dict(q=P + 4), ALIGN), (dict(out_head_stride=130), ALIGN),
    (dict(q_start=P + 2, max_q=2), ALIGN), (dict(out=P), ALIAS), (dict(work=None), ARG), (dict(work_bytes=16), SIZE),
    (dict(work=P + 8), ALIGN), (dict(scale=math.nan), ARG), (dict(scale=math.inf), ARG), (dict(n_tokens=1 << 29, n_seqs=1 << 29), SIZE),
    (dict(n_tokens=70000, n_seqs=70000), SIZE)])
def test_attn_refuses(kw, rc):
    assert attn(**kw) == rc


def test_attn_workspace_sizes():
    size = lambda **kw: Q.lib.q_b200_attn_work_bytes(C.byref(attn_args(**kw)))  # noqa: E731
    # one short sequence is done in one part
    assert size(max_prefix=0, max_len=8, n_seqs=1, n_tokens=1) == 0
    # parts of (o, m, l) in fp32 for each token's head
    need = size(work=None, work_bytes=0)
    assert need > 0 and need % (2 * 4 * (128 * 4 + 8)) == 0
    assert size(kv=cache(head_dim=80)) == 0


@pytest.mark.parametrize("kw,rc", [
    (dict(target=None), ARG), (dict(uniform=None), ARG), (dict(tokens=None), ARG), (dict(n_tokens=None), ARG),
    (dict(draft_tokens=None), ARG), (dict(dtype=3), DTYPE), (dict(kind=2), ARG), (dict(n_seqs=0), SIZE), (dict(vocab=0), SIZE),
    (dict(n_draft=32), SIZE), (dict(kind=1, temperature=-1.0), ARG), (dict(kind=1, temperature=math.nan), ARG),
    (dict(kind=1, temperature=math.inf), ARG), (dict(target=P + 2), ALIGN), (dict(uniform=P + 2), ALIGN), (dict(tokens=3 * P), ALIAS)])
def test_verify_refuses(kw, rc):
    assert verify(**kw) == rc


def test_batch_view_refuses():
    ctx, kv, pages, n = Q.q_context(), Q.q_b200_paged_kv(), C.c_void_p(), C.c_uint32()
    f = Q.lib.q_b200_batch_kv_view
    assert f(None, 0, C.byref(kv), C.byref(pages), C.byref(n)) == ARG
    assert f(C.byref(ctx), 0, C.byref(kv), C.byref(pages), None) == ARG
    assert f(C.byref(ctx), 0, C.byref(kv), C.byref(pages), C.byref(n)) == ARG  # no batch


# ---- frequency plans ---------------------------------------------------------------------------------------------


def scale(kind, factor=8.0, low=1.0, high=4.0, length=8192.0, gain=0.0, reserved=0):
    return Q.q_b200_rope_scale(kind, reserved, factor, low, high, length, gain)


def test_plan_refuses():
    f, p = Q.lib.q_b200_rope_plan_init, Q.q_b200_rope_plan()
    assert f(None, 64, 0, 1e4, None) == ARG
    for rot in (0, 1, 63, 258):
        assert f(C.byref(p), rot, 0, 1e4, None) == SIZE
    assert f(C.byref(p), 64, 2, 1e4, None) == ARG
    for base in (1.0, 0.0, -5.0, math.inf, math.nan):
        assert f(C.byref(p), 64, 0, base, None) == ARG
    for s in (scale(4), scale(1, factor=0.0), scale(1, factor=math.nan), scale(2, low=4.0, high=4.0), scale(2, length=0.0),
              scale(3, low=0.0), scale(3, gain=-1.0), scale(1, reserved=1)):
        assert f(C.byref(p), 64, 0, 1e4, C.byref(s)) == ARG


@pytest.mark.parametrize("rot", [2, 48, 128, 256])
def test_plan_frequencies(rot):
    i = np.arange(rot // 2)
    f = 500000.0 ** (-2.0 * i / rot)
    turns = lambda p: np.array(p.turns[: rot // 2]) * 2 * math.pi  # noqa: E731
    near = lambda a, b: np.testing.assert_allclose(a, b, rtol=1e-14)  # noqa: E731  (a few roundings of 2^-53)
    near(turns(plan(rot, base=500000.0)), f)
    near(turns(plan(rot, base=500000.0, scale=scale(1, 4.0))), f / 4.0)
    got = turns(plan(rot, base=500000.0, scale=scale(2)))
    wave = 2 * math.pi / f
    for w, v, g in zip(wave, f, got):  # long waves slowed, short kept, between them linear in turns
        if w > 8192.0:
            want = v / 8.0
        elif w < 8192.0 / 4.0:
            want = v
        else:
            s = (8192.0 / w - 1.0) / 3.0
            want = (1 - s) * v / 8.0 + s * v
        near(g, want)
    p = plan(rot, base=500000.0, scale=scale(3, high=32.0))
    assert p.gain == np.float32(0.1 * math.log(8.0) + 1.0)
    got = turns(p)
    assert (got <= f * (1 + 1e-12)).all() and (got >= f / 8.0 * (1 - 1e-12)).all()
    near(got[0], f[0] if rot > 2 else got[0])
    slow = np.floor(rot * math.log(8192.0 / (1.0 * 2 * math.pi)) / (2 * math.log(500000.0))) + 2
    near(got[i >= slow], f[i >= slow] / 8.0)
    assert plan(rot, base=500000.0, scale=scale(3, high=32.0, gain=1.25)).gain == 1.25
