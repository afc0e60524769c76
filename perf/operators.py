"""Cases of the serving operators for drafted, batched decoding: what is measured and what it has to give.

Four operators that a serving loop runs one after the other on device buffers:

  rope    rotary positions: interleaved and half pair layouts, part of the head, plain and scaled frequencies
  append  new keys and values into a paged cache, rotated on the way, the queries rotated beside them
  attn    attention of a batch over a prefix that all its sequences share and over each one's own pages
  verify  drafted tokens accepted or replaced by the target's probabilities, from given random numbers

`run` computes them in plain torch where `own` is false and through the package's entry points where it is true.  Tensors
have the layouts that the entry points take: caches are pools of pages [page][layer][kv head][row][K | V], seen by one layer.
"""
import math
import sys

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}
LAYOUTS = {"interleaved": 0, "half": 1}
SCALINGS = {"plain": 0, "linear": 1, "banded": 2, "yarn": 3}
BASE = 500000.0
FACTOR, BAND_LOW, BAND_HIGH, YARN_SLOW, YARN_FAST, TRAINED = 8.0, 1.0, 4.0, 1.0, 32.0, 8192.0


def package():
    if "project-ia_b200" not in sys.path:
        sys.path.insert(0, "project-ia_b200")
    import qorus_b200
    return qorus_b200


# ---- the cases -----------------------------------------------------------------------------------------------------


def listed():
    return [
        # one decoded token's query heads at the 8B shape (the framework's own decode step holds them in 32 bits)
        dict(name="rope one token", op="rope", dtype="f32", tokens=1, heads=32, dim=128, rot=128, layout="interleaved", scaling="plain",
             far=8192, transpose=False),
        # a 2048-token prompt's query heads at the 8B shape, positions scaled for a longer context
        dict(name="rope prompt", op="rope", dtype="f32", tokens=2048, heads=32, dim=128, rot=128, layout="interleaved", scaling="banded",
             far=131072, transpose=False),
        # the direction back (keys taken out of one position before they enter another, or a gradient), part of the head, far
        dict(name="rope back, partial", op="rope", dtype="bf16", tokens=8191, heads=40, dim=128, rot=96, layout="half", scaling="yarn",
             far=1048576, transpose=True),
        # one decode step of 16 sequences at the 8B shape into 32-bit pages, as the batched decode has them
        dict(name="append decode step", op="append", dtype="f32", cache="f32", tokens=16, seqs=16, heads=32, kv_heads=8, dim=128, rot=128,
             layout="interleaved", scaling="plain", page_rows=32, rows=512, layers=2),
        # chunks of 7 prompts, 4093 tokens in all, into 16-bit pages
        dict(name="append prompts", op="append", dtype="bf16", cache="bf16", tokens=4093, seqs=7, heads=32, kv_heads=8, dim=128, rot=128,
             layout="half", scaling="banded", page_rows=64, rows=640, layers=1),
        # four sequences after a short shared instruction, one token each, in the batched decode's 32-bit cache
        dict(name="attn small f32", op="attn", dtype="f32", seqs=4, max_q=1, ragged=False, pad=0, heads=32, kv_heads=8, dim=128,
             page_rows=32, prefix=512, rows=130, layers=2, short=False),
        # sixteen sequences after a shared prompt, one token each
        dict(name="attn decode bf16", op="attn", dtype="bf16", seqs=16, max_q=1, ragged=False, pad=0, heads=32, kv_heads=8, dim=128,
             page_rows=64, prefix=4096, rows=1024, layers=1, short=False),
        # up to five drafted tokens of sixteen sequences scored at once, narrow heads, pages that end inside a tile
        dict(name="attn drafts f16", op="attn", dtype="f16", seqs=16, max_q=5, ragged=True, pad=3, heads=32, kv_heads=8, dim=64,
             page_rows=48, prefix=8190, rows=777, layers=1, short=True),
        # a wide batch at the 70B shape over a long shared document
        dict(name="attn wide bf16", op="attn", dtype="bf16", seqs=64, max_q=1, ragged=False, pad=0, heads=64, kv_heads=8, dim=128,
             page_rows=64, prefix=32768, rows=512, layers=1, short=False),
        # one sequence with four drafted tokens, probabilities over the whole vocabulary
        dict(name="verify one", op="verify", kind="probs", dtype="f32", seqs=1, drafts=4, vocab=128256, temperature=1.0, apart=0.5),
        # a wide batch, probabilities kept in 16 bits
        dict(name="verify batch", op="verify", kind="probs", dtype="bf16", seqs=64, drafts=7, vocab=128256, temperature=1.0, apart=0.5),
        # logits as the batched decode step leaves them, at a temperature
        dict(name="verify logits", op="verify", kind="logits", dtype="f32", seqs=16, drafts=4, vocab=128256, temperature=0.8, apart=0.5),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rope", "append", "attn", "attn", "verify"])
    if op == "rope":
        dim = rng.choice([32, 64, 80, 128, 256])
        heads = rng.randint(1, 64)
        dtype = rng.choice(["f32", "f16", "bf16"])
        tokens = min(_log(rng, 1, 16384), 84_000_000 // (heads * dim * _bytes(dtype)))
        return dict(op=op, dtype=dtype, tokens=tokens, heads=heads, dim=dim,
                    rot=rng.choice([dim, dim // 2, 2 * rng.randint(1, dim // 2)]), layout=rng.choice(["interleaved", "half"]),
                    scaling=rng.choice(["plain", "linear", "banded", "yarn"]), far=_log(rng, 64, 1048576), transpose=rng.random() < 0.3)
    if op == "append":
        dim, kv_heads = rng.choice([32, 64, 128]), rng.choice([1, 2, 5, 8])
        seqs, heads = rng.randint(1, 64), kv_heads * rng.choice([0, 1, 4, 8])
        tokens = min(_log(rng, 1, 8192), 12_000_000 // ((heads + 2 * kv_heads) * dim))
        return dict(op=op, dtype=rng.choice(["f32", "f16", "bf16"]), cache=rng.choice(["f32", "f16", "bf16"]), tokens=tokens, seqs=seqs,
                    heads=heads, kv_heads=kv_heads, dim=dim, rot=rng.choice([0, dim, dim // 2]),
                    layout=rng.choice(["interleaved", "half"]), scaling=rng.choice(["plain", "linear", "banded", "yarn"]),
                    page_rows=rng.choice([16, 17, 32, 48, 64, 128]), rows=-(-tokens // seqs) + rng.randint(0, 100), layers=rng.choice([1, 2]))
    if op == "attn":
        kv_heads, group, dim = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 7, 8]), rng.choice([32, 64, 128])
        max_q = rng.choice([1, 1, 1, _log(rng, 1, 8), _log(rng, 2, 128)])
        seqs = max(1, min(_log(rng, 1, 64), 256 // max_q))
        dtype = rng.choice(["f32", "f16", "bf16"])
        rows = _log(rng, max(2, max_q), (512 if seqs > 16 else 2048) // (2 if dtype == "f32" else 1))
        longest = (32768 if seqs * max_q * group <= 256 else 4096) // (2 if dtype == "f32" else 1)
        return dict(op=op, dtype=dtype, seqs=seqs, max_q=max_q, ragged=max_q > 1 and rng.random() < 0.6,
                    pad=rng.choice([0, 0, 3]), heads=kv_heads * group, kv_heads=kv_heads, dim=dim, page_rows=rng.choice([16, 17, 32, 48, 64, 128]),
                    prefix=0 if rng.random() < 0.1 else _log(rng, 1, longest), rows=rows,
                    layers=rng.choice([1, 2]), short=rng.random() < 0.3)
    seqs, drafts = _log(rng, 1, 64), rng.randint(1, 7)
    vocab = min(_log(rng, 259, 128256), 48_000_000 // (seqs * (2 * drafts + 1)))
    return dict(op=op, kind=rng.choice(["probs", "logits"]), dtype=rng.choice(["f32", "f16", "bf16"]), seqs=seqs, drafts=drafts, vocab=vocab,
                temperature=rng.choice([0.0, 0.6, 0.8, 1.0, 1.3]), apart=rng.choice([0.1, 0.5, 1.0]))


def _bytes(dtype):
    return 4 if dtype == "f32" else 2


def _spread(n, low, high, step):
    """n whole numbers over [low, high], the same for every seed, so that a case's work is known."""
    return [low + int((high - low + 0.999) * math.modf((b + 1) * step)[0]) for b in range(n)]


def _counts(case):
    """New tokens and own rows (the new ones among them) of each sequence of an attention case."""
    new = _spread(case["seqs"], 1, case["max_q"], 0.381966) if case["ragged"] else [case["max_q"]] * case["seqs"]
    rows = [max(n, r) for n, r in zip(new, _spread(case["seqs"], 1, case["rows"], 0.618034))]
    if case["short"]:
        rows[0] = 0  # a sequence that has nothing but the prefix yet
    return new, rows


def work(case):
    c = case
    if c["op"] == "rope":
        n = c["tokens"] * c["heads"]
        return {"bytes": 2 * n * c["dim"] * _bytes(c["dtype"]) + 4 * c["tokens"], "flops": 3 * n * c["rot"]}
    if c["op"] == "append":
        kv = 2 * c["kv_heads"] * c["dim"]
        return {"bytes": c["tokens"] * (kv * (_bytes(c["dtype"]) + _bytes(c["cache"])) + 2 * c["heads"] * c["dim"] * _bytes(c["dtype"]) + 12),
                "flops": 3 * c["tokens"] * (c["heads"] + c["kv_heads"]) * c["rot"]}
    if c["op"] == "attn":
        new, rows = _counts(c)
        seen = sum(n * c["prefix"] + sum(max(0, r - n + 1 + i) for i in range(n)) for n, r in zip(new, rows))
        return {"bytes": _bytes(c["dtype"]) * (2 * c["kv_heads"] * c["dim"] * (c["prefix"] + sum(rows)) + 2 * sum(new) * c["heads"] * c["dim"]),
                "flops": 4 * c["dim"] * c["heads"] * seen}
    # probabilities: the row that the token is drawn from, and the draft's beside it; logits: every drafted row's sum too
    rows = c["seqs"] * (2 * c["drafts"] if c["kind"] == "logits" and c["temperature"] > 0 else c["drafts"] if c["kind"] == "logits" else 2)
    return {"bytes": rows * c["vocab"] * _bytes(c["dtype"]), "flops": 4 * rows * c["vocab"]}


# ---- inputs --------------------------------------------------------------------------------------------------------


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 13)
    return g


def _frequencies(rot, scaling):
    """Angle of one position for each pair, in 64 bits, and the factor on cosine and sine."""
    i = torch.arange(rot // 2, dtype=torch.float64)
    f = BASE ** (-2.0 * i / rot)
    if scaling == "linear":
        return f / FACTOR, 1.0
    if scaling == "banded":  # long waves slowed down, short ones kept, a ramp between
        s = ((TRAINED * f / (2 * math.pi) - BAND_LOW) / (BAND_HIGH - BAND_LOW)).clamp(0.0, 1.0)
        return (1 - s) * f / FACTOR + s * f, 1.0
    if scaling == "yarn":  # the ramp over the pairs' indexes
        at = lambda turns: rot * math.log(TRAINED / (turns * 2 * math.pi)) / (2 * math.log(BASE))  # noqa: E731
        low, high = max(math.floor(at(YARN_FAST)), 0), min(math.ceil(at(YARN_SLOW)), rot - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        return f / FACTOR * ramp + f * (1 - ramp), 0.1 * math.log(FACTOR) + 1.0
    return f, 1.0


def _plan(case):
    """The rotation's plan, as a program keeps it beside its model."""
    if not own or not case["rot"]:
        return None
    Q = package()
    plan = Q.q_b200_rope_plan()
    scale = Q.q_b200_rope_scale(SCALINGS[case["scaling"]], 0, FACTOR, BAND_LOW if case["scaling"] == "banded" else YARN_SLOW,
                                BAND_HIGH if case["scaling"] == "banded" else YARN_FAST, TRAINED, 0.0)
    Q.check(Q.lib.q_b200_rope_plan_init(Q.C.byref(plan), case["rot"], LAYOUTS[case["layout"]], BASE, Q.C.byref(scale)), "q_b200_rope_plan_init")
    return plan


def _pool(case, pages, dtype, g):
    """A pool of pages, and one layer's keys and values in it: [page][kv head][row][dim] each."""
    shape = (max(1, pages), case["layers"], case["kv_heads"], case["page_rows"], 2 * case["dim"])
    pool = torch.randn(shape, device="cuda", generator=g, dtype=torch.float32 if dtype == "f32" else torch.float16).to(DTYPES[dtype])
    return pool, pool[:, -1, :, :, : case["dim"]], pool[:, -1, :, :, case["dim"]:]


def prepare(case, seed):
    c, g = case, _generator(seed)
    dev = dict(device="cuda")
    normal = lambda *s: torch.randn(s, generator=g, **dev)  # noqa: E731
    if c["op"] == "rope":
        x = normal(c["tokens"], c["heads"], c["dim"]).to(DTYPES[c["dtype"]])
        pos = torch.randint(0, c["far"], (c["tokens"],), generator=g, dtype=torch.int32, **dev)
        f, gain = _frequencies(c["rot"], c["scaling"])
        return dict(case=c, x=x, out=torch.empty_like(x), pos=pos, f=f.cuda(), gain=gain, plan=_plan(c))
    if c["op"] == "append":
        per = -(-c["rows"] // c["page_rows"])
        pool, keys, values = _pool(c, c["seqs"] * per, c["cache"], g)
        pages = torch.randperm(c["seqs"] * per, generator=g, **dev).to(torch.int32).view(c["seqs"], per)
        t = torch.arange(c["tokens"], **dev)
        seq, row = t % c["seqs"], t // c["seqs"]
        row = (row + (c["rows"] - 1 - row.max())).to(torch.int32)  # the last rows of each sequence's pages
        row[-1] = -1 if c["tokens"] > 1 else row[-1]  # a padded token, which leaves everything as it is
        pos = row + torch.randint(0, 4096, (1,), generator=g, dtype=torch.int32, **dev)  # behind a prefix that has its own pages
        # what a fused projection leaves: queries, keys and values of a token in one row
        qkv = normal(c["tokens"], (c["heads"] + 2 * c["kv_heads"]) * c["dim"]).to(DTYPES[c["dtype"]])
        a, b = c["heads"] * c["dim"], (c["heads"] + c["kv_heads"]) * c["dim"]
        f, gain = _frequencies(c["rot"], c["scaling"]) if c["rot"] else (None, 1.0)
        st = dict(case=c, pool=pool, keys=keys, values=values, pages=pages, seq=seq.to(torch.int32), row=row, pos=pos,
                  q=qkv[:, :a].view(c["tokens"], c["heads"], c["dim"]), k=qkv[:, a:b].view(c["tokens"], c["kv_heads"], c["dim"]),
                  v=qkv[:, b:].view(c["tokens"], c["kv_heads"], c["dim"]), f=None if f is None else f.cuda(), gain=gain, plan=_plan(c))
        st["out"] = torch.zeros(c["tokens"], c["heads"], c["dim"], dtype=DTYPES[c["dtype"]], **dev)
        return st
    if c["op"] == "attn":
        new, rows = _counts(c)
        n, R = sum(new), c["page_rows"]
        per, shared = -(-max(rows + [1]) // R), -(-c["prefix"] // R)
        pool, keys, values = _pool(c, c["seqs"] * per + shared, c["dtype"], g)
        ids = torch.randperm(c["seqs"] * per + shared, generator=g, **dev).to(torch.int32)
        q = (normal(n + c["pad"], c["heads"], c["dim"]) * 2.0).to(DTYPES[c["dtype"]])
        start = torch.tensor([0] + new, dtype=torch.int32).cumsum(0).to(torch.int32)
        seq = torch.repeat_interleave(torch.arange(c["seqs"]), torch.tensor(new))
        return dict(case=c, keys=keys, values=values, q=q, out=torch.zeros_like(q), pages=ids[shared:].view(c["seqs"], per), prefix_pages=ids[:shared],
                    prefix_len=torch.tensor([c["prefix"]], dtype=torch.int32, **dev), lens=torch.tensor(rows, dtype=torch.int32, **dev),
                    start=start.cuda(), seq=seq.cuda(), nth=(torch.arange(n) - start[:-1].long()[seq]).cuda(), new=torch.tensor(new, **dev),
                    tokens=n, max_len=max(rows), work=None)
    S, K, V, T = c["seqs"], c["drafts"], c["vocab"], c["temperature"] or 1.0
    target = normal(S, K + 1, V) * 3.0
    draft = target[:, :K] + normal(S, K, V) * c["apart"]
    noise = torch.rand(S, K, V, generator=g, **dev)
    tokens = (draft / T - torch.log(-torch.log(noise))).argmax(-1).to(torch.int32)
    del noise
    if c["kind"] == "probs":
        target, draft = torch.softmax(target / T, -1), torch.softmax(draft / T, -1)
    length = torch.tensor(_spread(S, max(1, K - 1), K, 0.618034), dtype=torch.int32, **dev)  # some were drafted one token less
    return dict(case=c, target=target.to(DTYPES[c["dtype"]]), draft=draft.to(DTYPES[c["dtype"]]), tokens=tokens, length=length,
                uniform=torch.rand(S, K + 1, generator=g, **dev), chosen=torch.zeros(S, K + 1, dtype=torch.int32, **dev),
                count=torch.zeros(S, dtype=torch.int32, **dev))


# ---- the plain forms -----------------------------------------------------------------------------------------------


def _rotated(x, pos, f, gain, rot, layout, back=False):
    """x [tokens][heads][dim] turned by its positions, in 32 bits; the angles in 64."""
    angle = pos.to(torch.float64)[:, None] * f
    cos = (angle.cos() * gain).float()[:, None]
    sin = (angle.sin() * (-gain if back else gain)).float()[:, None]
    y = x.float().clone()
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if layout == "interleaved" else (y[..., : rot // 2], y[..., rot // 2: rot])
    a1, b1 = a * cos - b * sin, a * sin + b * cos
    a.copy_(a1)
    b.copy_(b1)
    return y


def _plain_rope(s):
    c = s["case"]
    s["out"].copy_(_rotated(s["x"], s["pos"], s["f"], s["gain"], c["rot"], c["layout"], c["transpose"]).to(s["out"].dtype))
    return s["out"]


def _plain_append(s):
    c = s["case"]
    live = (s["row"] >= 0).nonzero()[:, 0]
    row, pos = s["row"][live].long(), s["pos"][live]
    page = s["pages"][s["seq"][live].long(), row // c["page_rows"]].long()
    k, q = s["k"][live].float(), s["q"][live].float()
    if c["rot"]:
        k = _rotated(k, pos, s["f"], s["gain"], c["rot"], c["layout"])
        q = _rotated(q, pos, s["f"], s["gain"], c["rot"], c["layout"])
    s["keys"].permute(0, 2, 1, 3)[page, row % c["page_rows"]] = k.to(s["keys"].dtype)
    s["values"].permute(0, 2, 1, 3)[page, row % c["page_rows"]] = s["v"][live].float().to(s["keys"].dtype)
    s["out"][live] = q.to(s["out"].dtype)
    return s["pool"], s["out"]


def _rows_of(t, pages):
    """[kv head][row][dim] of the rows that a list of pages (or lists of them, in front) holds."""
    x = t[pages.long()].float()
    x = x.movedim(-4, -3).flatten(-3, -2)
    return x


def _plain_attn(s):
    c = s["case"]
    B, M, KV, G, D, P = c["seqs"], c["max_q"], c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"], c["prefix"]
    scale = 1.0 / math.sqrt(D)
    q = s["q"][: s["tokens"]].float().view(-1, KV, G, D)
    mat = torch.zeros(B, M, KV, G, D, device="cuda")
    mat[s["seq"], s["nth"]] = q
    k_own, v_own = _rows_of(s["keys"], s["pages"]), _rows_of(s["values"], s["pages"])  # [seq][kv head][row][dim]
    own_s = torch.einsum("bmkgd,bkld->bkgml", mat, k_own) * scale
    last = s["lens"].long()[:, None] - s["new"][:, None] + torch.arange(M, device="cuda")  # last row that the m-th new token sees
    seen = torch.arange(k_own.shape[2], device="cuda") <= last[..., None]
    own_s = own_s.masked_fill(~seen[:, None, None], -math.inf)
    own_s = own_s.permute(0, 3, 1, 2, 4)[s["seq"], s["nth"]]  # [token][kv head][g][row]
    top = own_s.amax(-1)
    if P:
        k_all, v_all = _rows_of(s["keys"], s["prefix_pages"])[:, :P], _rows_of(s["values"], s["prefix_pages"])[:, :P]
        all_s = torch.matmul(q.permute(1, 0, 2, 3).reshape(KV, -1, D), k_all.transpose(1, 2)) * scale
        all_s = all_s.view(KV, -1, G, P).permute(1, 0, 2, 3)
        top = torch.maximum(top, all_s.amax(-1))
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)[..., None]
    own_p = torch.exp(own_s - top)
    total = own_p.sum(-1)
    mat_p = torch.zeros(B, M, KV, G, own_p.shape[-1], device="cuda")
    mat_p[s["seq"], s["nth"]] = own_p
    out = torch.einsum("bmkgl,bkld->bmkgd", mat_p, v_own)[s["seq"], s["nth"]]
    if P:
        all_p = torch.exp(all_s - top)
        total = total + all_p.sum(-1)
        out = out + torch.matmul(all_p.permute(1, 0, 2, 3).reshape(KV, -1, P), v_all).view(KV, -1, G, D).permute(1, 0, 2, 3)
    out = torch.where(total[..., None] > 0, out / total[..., None].clamp_min(1e-37), torch.zeros_like(out))
    s["out"][: s["tokens"]] = out.reshape(-1, c["heads"], D).to(s["out"].dtype)
    return s["out"]


def _weights(x, case):
    """Probabilities in 64 bits of rows of probabilities or logits: values next to a border decide a whole token."""
    x = x.double()
    if case["kind"] == "probs":
        return x
    if case["temperature"] < 1e-6:
        return torch.zeros_like(x).scatter_(-1, x.argmax(-1, keepdim=True), 1.0)
    e = torch.exp((x - x.amax(-1, keepdim=True)) / float(np.float32(case["temperature"])))
    return e / e.sum(-1, keepdim=True)


def _plain_verify(s):
    c = s["case"]
    S, K = s["tokens"].shape
    at, x = torch.arange(S, device="cuda"), s["tokens"].long()
    if c["kind"] == "probs":
        p = s["target"][:, :K].gather(-1, x[..., None])[..., 0].double()
        q = s["draft"].gather(-1, x[..., None])[..., 0].double()
    else:
        p = _weights(s["target"][:, :K], c).gather(-1, x[..., None])[..., 0]
        q = _weights(s["draft"], c).gather(-1, x[..., None])[..., 0]
    if c["kind"] == "logits" and c["temperature"] < 1e-6:
        q = torch.ones_like(p)  # greedy: the drafted token is the target's own or it is not
    i = torch.arange(K, device="cuda")
    fine = (s["uniform"][:, :K].double() * q < p) & (i < s["length"][:, None])
    n = fine.long().cumprod(-1).sum(-1)
    w = _weights(s["target"][at, n], c)
    less = _weights(s["draft"][at, n.clamp_max(K - 1)], c)
    if c["kind"] == "logits" and c["temperature"] < 1e-6:
        less = torch.zeros_like(less)
    rest = torch.where((n < s["length"])[:, None], w - less, w).clamp_min(0.0)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, w)
    total = rest.cumsum(-1)
    reached = total > s["uniform"][:, K:].double() * total[:, -1:]
    v = torch.arange(rest.shape[-1], device="cuda")
    last = torch.where(rest > 0, v, torch.zeros_like(v)).amax(-1)
    token = torch.where(reached.any(-1), reached.byte().argmax(-1), last)
    slot = torch.arange(K + 1, device="cuda")
    drafted = torch.nn.functional.pad(x, (0, 1))
    s["chosen"].copy_(torch.where(slot < n[:, None], drafted, torch.where(slot == n[:, None], token[:, None], torch.full_like(drafted, -1))))
    s["count"].copy_(n + 1)
    return s["chosen"], s["count"]


# ---- the calls of the package --------------------------------------------------------------------------------------


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _cache(Q, s, dtype):
    k, v, c = s["keys"], s["values"], s["case"]
    return Q.q_b200_paged_kv(k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), k.stride(2), k.shape[0], c["page_rows"], c["kv_heads"], c["dim"],
                             CODES[dtype], 0)


def _own_rope(s):
    Q, c, x, out = package(), s["case"], s["x"], s["out"]
    args = Q.q_b200_rope_args(x.data_ptr(), out.data_ptr(), s["pos"].data_ptr(), Q.C.addressof(s["plan"]), x.stride(0), x.stride(1), out.stride(0),
                              out.stride(1), c["tokens"], c["heads"], c["dim"], CODES[c["dtype"]], int(c["transpose"]), 0)
    Q.check(Q.lib.q_b200_rope(Q.C.byref(args), _stream()), "q_b200_rope")
    return out


def _own_append(s):
    Q, c, q, k, v, out = package(), s["case"], s["q"], s["k"], s["v"], s["out"]
    args = Q.q_b200_append_args(_cache(Q, s, c["cache"]), k.data_ptr(), v.data_ptr(), q.data_ptr() if c["heads"] else None,
                                out.data_ptr() if c["heads"] else None, k.stride(0), k.stride(1), v.stride(0), v.stride(1), q.stride(0), q.stride(1),
                                out.stride(0), out.stride(1), s["pages"].data_ptr(), s["seq"].data_ptr(), s["row"].data_ptr(), s["pos"].data_ptr(),
                                Q.C.addressof(s["plan"]) if c["rot"] else None, c["tokens"], c["seqs"], s["pages"].shape[1], c["heads"],
                                CODES[c["dtype"]], 0)
    Q.check(Q.lib.q_b200_kv_append(Q.C.byref(args), _stream()), "q_b200_kv_append")
    return s["pool"], out


def _own_attn(s):
    Q, c, q, out = package(), s["case"], s["q"], s["out"]
    args = Q.q_b200_attn_args(_cache(Q, s, c["dtype"]), q.data_ptr(), out.data_ptr(), q.stride(0), q.stride(1), out.stride(0), out.stride(1),
                              s["start"].data_ptr() if c["max_q"] > 1 else None, s["pages"].data_ptr(), s["lens"].data_ptr(),
                              s["prefix_pages"].data_ptr() if c["prefix"] else None, s["prefix_len"].data_ptr() if c["prefix"] else None, None, 0,
                              q.shape[0] if c["max_q"] > 1 else c["seqs"], c["seqs"], c["heads"], s["pages"].shape[1], c["max_q"], s["max_len"],
                              c["prefix"], 1.0 / math.sqrt(c["dim"]))
    if s["work"] is None:  # the workspace, which a program keeps for all its layers
        s["work"] = torch.empty(max(16, Q.lib.q_b200_attn_work_bytes(Q.C.byref(args))), dtype=torch.uint8, device="cuda")
    args.work, args.work_bytes = s["work"].data_ptr(), s["work"].numel()
    Q.check(Q.lib.q_b200_attn_prefix(Q.C.byref(args), _stream()), "q_b200_attn_prefix")
    return out


def _own_verify(s):
    Q, c, t, d = package(), s["case"], s["target"], s["draft"]
    args = Q.q_b200_verify_args(t.data_ptr(), d.data_ptr(), t.stride(0), t.stride(1), d.stride(0), d.stride(1), s["tokens"].data_ptr(),
                                s["length"].data_ptr(), s["uniform"].data_ptr(), s["chosen"].data_ptr(), s["count"].data_ptr(), c["seqs"],
                                c["drafts"], c["vocab"], CODES[c["dtype"]], int(c["kind"] == "logits"), c["temperature"])
    Q.check(Q.lib.q_b200_verify_draft(Q.C.byref(args), _stream()), "q_b200_verify_draft")
    return s["chosen"], s["count"]


PLAIN = {"rope": _plain_rope, "append": _plain_append, "attn": _plain_attn, "verify": _plain_verify}
OWN = {"rope": _own_rope, "append": _own_append, "attn": _own_attn, "verify": _own_verify}


def run(state):
    return (OWN if own else PLAIN)[state["case"]["op"]](state)


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------


def _turned(x, pos, case, back=False):
    """Each pair as a complex number, times e^(i angle)."""
    rot = case["rot"]
    x = x.double().clone()
    if not rot:
        return x
    f, gain = _frequencies(rot, case["scaling"])
    turn = torch.polar(torch.full((len(pos), rot // 2), gain, dtype=torch.float64, device="cuda"),
                       pos.double()[:, None] * f.cuda() * (-1.0 if back else 1.0))[:, None]
    if case["layout"] == "interleaved":
        z = torch.complex(x[..., 0:rot:2].contiguous(), x[..., 1:rot:2].contiguous()) * turn
        x[..., 0:rot:2], x[..., 1:rot:2] = z.real, z.imag
    else:
        z = torch.complex(x[..., : rot // 2].contiguous(), x[..., rot // 2: rot].contiguous()) * turn
        x[..., : rot // 2], x[..., rot // 2: rot] = z.real, z.imag
    return x


def _exact_append(c, s):
    pool, out = s["pool"].double(), s["out"].double()
    k, q, v = _turned(s["k"], s["pos"], c), _turned(s["q"], s["pos"], c), s["v"].double()
    row, seq, pages = (s[n].cpu().tolist() for n in ("row", "seq", "pages"))
    live = [t for t in range(c["tokens"]) if row[t] >= 0]
    at = torch.tensor([pages[seq[t]][row[t] // c["page_rows"]] for t in live], device="cuda")
    within = torch.tensor([row[t] % c["page_rows"] for t in live], device="cuda")
    live = torch.tensor(live, device="cuda")
    for h in range(c["kv_heads"]):
        pool[at, -1, h, within] = torch.cat([k[live, h], v[live, h]], -1)
    out[live] = q[live]
    return pool, out


def _exact_attn(c, s):
    out = s["out"].double()
    D, G = c["dim"], c["heads"] // c["kv_heads"]
    new, rows = _counts(c)
    at = 0
    for b in range(c["seqs"]):
        n, r = new[b], rows[b]
        for h in range(c["kv_heads"]):
            k = torch.cat([s["keys"][:, h][s["prefix_pages"].long()].reshape(-1, D)[: c["prefix"]], s["keys"][:, h][s["pages"][b].long()].reshape(-1, D)[:r]])
            v = torch.cat([s["values"][:, h][s["prefix_pages"].long()].reshape(-1, D)[: c["prefix"]], s["values"][:, h][s["pages"][b].long()].reshape(-1, D)[:r]])
            q = s["q"][at: at + n, h * G: (h + 1) * G].double()
            score = torch.einsum("ngd,ld->ngl", q, k.double()) / math.sqrt(D)
            j = torch.arange(len(k), device="cuda") - c["prefix"]  # own row; the prefix, below zero, is in everyone's sight
            hidden = (j >= 0) & (j > r - n + torch.arange(n, device="cuda")[:, None])
            p = torch.softmax(score.masked_fill(hidden[:, None], -math.inf), -1)
            out[at: at + n, h * G: (h + 1) * G] = torch.einsum("ngl,ld->ngd", torch.nan_to_num(p), v.double())
        at += n
    return out


def _exact_verify(c, s):
    S, K, V = c["seqs"], c["drafts"], c["vocab"]
    chosen, count = np.full((S, K + 1), -1, np.int32), np.zeros(S, np.int32)
    length, u, x = s["length"].cpu().numpy(), s["uniform"].double().cpu().numpy(), s["tokens"].cpu().numpy()

    def law(row):
        row = row.double().cpu().numpy()
        if c["kind"] == "probs":
            return row
        if c["temperature"] < 1e-6:
            return (np.arange(V) == row.argmax()).astype(np.float64)
        e = np.exp((row - row.max()) / float(np.float32(c["temperature"])))
        return e / e.sum()

    greedy = c["kind"] == "logits" and c["temperature"] < 1e-6
    for b in range(S):
        n, q = 0, None
        while n < length[b]:
            p, q = law(s["target"][b, n]), law(s["draft"][b, n])
            if not u[b, n] * (1.0 if greedy else q[x[b, n]]) < p[x[b, n]]:
                break
            chosen[b, n] = x[b, n]
            n += 1
        p = law(s["target"][b, n])
        rest = np.maximum(p - q, 0.0) if n < length[b] and not greedy else p
        rest = rest if rest.sum() > 0 else p
        total = np.cumsum(rest)
        v = int(np.searchsorted(total, u[b, K] * total[-1], side="right"))
        chosen[b, n] = v if v < V else int(np.flatnonzero(rest)[-1])
        count[b] = n + 1
    return chosen, count


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _turned(s["x"], s["pos"], case, case["transpose"])
    return {"append": _exact_append, "attn": _exact_attn, "verify": _exact_verify}[case["op"]](case, s)
