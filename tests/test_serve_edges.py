"""Argument checks and plans of the serving operators at their limits, without a GPU (helpers: test_serve.py)."""
import ctypes as C
import math

import numpy as np
import pytest

import qorus_b200 as Q
from test_serve import ALIAS, ARG, P, SIZE, attn, attn_args, cache, plan, scale, verify


def work_bytes(**kw):
    return Q.lib.q_b200_attn_work_bytes(C.byref(attn_args(**kw)))


# ---- sizes whose products pass 2^64, or the grid ---------------------------------------------------------------------


@pytest.mark.parametrize("kw", [
    dict(n_seqs=1 << 31, max_q=1 << 31, n_heads=4, kv=cache(n_kv_heads=4)),  # 2^64
    dict(n_seqs=1 << 31, max_q=1 << 30, n_heads=8), dict(n_seqs=1 << 16, max_q=1 << 16, n_heads=1 << 31),
    dict(n_seqs=0xFFFFFFFF, max_q=0xFFFFFFFF, n_heads=0xFFFFFFFE), dict(n_seqs=1, max_q=1 << 30, n_heads=2),
    dict(n_tokens=0xFFFFFFFF, n_seqs=1, n_heads=0xFFFFFFFE)])
def test_attn_products_of_sizes_do_not_wrap(kw):
    kw = dict(dict(q_start=8 * P, n_tokens=2), **kw)
    assert work_bytes(**kw) == 0
    assert attn(**kw) == SIZE


@pytest.mark.parametrize("kw", [
    dict(n_tokens=70000, n_seqs=70000, n_heads=2),                              # own rows: a tile for each sequence
    dict(n_tokens=70000, n_seqs=1000, max_q=70, n_heads=128, q_start=8 * P),    # 70 tiles for each of 1000
    dict(n_tokens=4_194_241, n_seqs=2, max_q=8, n_heads=2, q_start=8 * P)])     # the prefix: 65536 tiles of 64 for all tokens
def test_attn_work_bytes_is_zero_where_the_call_is_refused(kw):
    kw = dict(kw, kv=cache(n_kv_heads=2))
    assert work_bytes(**kw) == 0
    assert attn(**kw) == SIZE


# ---- outputs that lie over what is still read ------------------------------------------------------------------------


@pytest.mark.parametrize("kw,rc", [  # 2 sequences of 4 drafts: tokens and uniform 40 bytes, draft_tokens 32, the others 8
    (dict(tokens=3 * P + 28), ALIAS), (dict(tokens=3 * P - 36), ALIAS), (dict(tokens=3 * P + 32), ARG), (dict(tokens=3 * P - 40), ARG),
    (dict(tokens=4 * P), ALIAS), (dict(tokens=4 * P + 36), ALIAS), (dict(tokens=4 * P + 40), ARG),
    (dict(n_tokens=3 * P + 16), ALIAS), (dict(n_tokens=4 * P + 12), ALIAS), (dict(n_tokens=5 * P + 36), ALIAS),
    (dict(n_tokens=5 * P + 40), ARG), (dict(n_tokens=5 * P - 4), ALIAS), (dict(n_tokens=5 * P - 8), ARG),
    (dict(draft_len=7 * P, tokens=7 * P + 4), ALIAS), (dict(draft_len=7 * P, n_tokens=7 * P), ALIAS), (dict(draft_len=7 * P, n_tokens=7 * P + 8), ARG)])
def test_verify_refuses_outputs_over_its_inputs(kw, rc):
    # ARG: no overlap, so the refusal is the one of pointers that are no device memory
    assert verify(**kw) == rc


# ---- plans -----------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("seqs,new,prefix,rows", [(32, 4, 16384, 256), (24, 4, 16384, 256), (32, 4, 8192, 64)])
def test_attn_prefix_gets_the_sms_that_its_work_asks_for(seqs, new, prefix, rows):
    # bf16, 32/8 heads of 128: 16 CTAs for each part of the prefix, whose work is 0.85 of the whole or more.  The own rows (8 splits
    # of a cluster at most) leave nothing in the workspace, so its parts are the prefix's: as many as the 148 SMs run at once.
    kw = dict(n_tokens=seqs * new, n_seqs=seqs, max_q=new, n_heads=32, max_prefix=prefix, max_len=rows, q_start=8 * P, pages_per_seq=rows // 32,
              kv=cache(n_kv_heads=8, dtype=Q.Q_B200_BF16))
    parts, rest = divmod(work_bytes(**kw), seqs * new * 32 * (128 * 4 + 8))
    assert rest == 0 and 0.85 * 148 <= parts * 16 <= 148


# ---- frequencies -----------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("rot", [2, 6, 48, 128, 256])
@pytest.mark.parametrize("base", [10000.0, 500000.0])
@pytest.mark.parametrize("factor,low,high,length", [
    (8.0, 1.0, 32.0, 8192.0), (4.0, 1.0, 32.0, 4096.0), (40.0, 0.5, 3.0, 1000.0),
    (16.0, 1.0, 1.5, 131072.0),                                # a ramp of a pair or two
    (2.0, 1.0, 32.0, 50.0),                                    # every wave turns less than 32 times: the ramp begins before pair 0
    (2.0, 1e-9, 1e-8, 4096.0), (0.5, 1.0, 32.0, 1e30)])        # it ends behind the last pair; every pair turns more than that
def test_yarn_frequencies_pair_by_pair(rot, base, factor, low, high, length):
    p = plan(rot, base=base, scale=scale(3, factor, low, high, length))
    # the pair (a fraction) whose wave turns n times in `length` positions: n 2 pi = length base^(-2i/rot)
    pair = lambda n: rot / 2 * math.log(length / (2 * math.pi * n), base)  # noqa: E731
    ends = [pair(high), pair(low)]
    if any(abs(e - round(e)) < 1e-9 * max(1.0, abs(e)) for e in ends):
        pytest.skip("an end on a pair: a matter of rounding")
    first, last = max(math.floor(ends[0]), 0), min(math.ceil(ends[1]), rot - 1)
    for i in range(rot // 2):
        f = base ** (-2 * i / rot)
        kept = 1.0 - min(max((i - first) / max(last - first, 0.001), 0.0), 1.0)
        want = kept * f + (1.0 - kept) * f / factor
        # roundings of 2^-53: the power's (its exponent's times ln base < 14), a dozen others
        assert abs(p.turns[i] * 2 * math.pi - want) <= 1e-14 * want, i
    assert p.gain == np.float32(0.1 * math.log(factor) + 1.0) and p.rot_dim == rot
