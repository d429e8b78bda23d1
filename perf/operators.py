"""What the operators for several continuations of one prompt are timed on.

Four kinds of work:

  attend   `hira_shared_attention`: decode attention of a batch whose sequences ("branches") share their
           prompts; each prompt's keys and values serve all its branches, each branch has a tail of its own
  select   `CUDAIndexer.select`: the sequences of an index forked or compacted into a new index
  reorder  `CUDAIndexer.reorder` and `SharedPrompt.reorder`: sequences replaced in place by others, as a
           search over continuations does after each step
  rotate   `hira_qk_norm_rope`: norms of the query and key heads and the position rotation in one pass

`own` is set from outside: False runs the operators in their plain form (elementary torch operations in 32
bits), True the framework's.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-6
ROPE_BASE = 500000.0


def _attend(name, *, prompts=1, branches=16, kv=8, group=4, dim=128, dtype="bf16", ctx=32768, tail=64, lq=1, ragged=False):
    c = {"kind": "attend", "prompts": prompts, "branches": branches, "kv": kv, "group": group, "dim": dim, "dtype": dtype,
         "ctx": ctx, "tail": tail, "lq": lq, "ragged": ragged}
    return c if name is None else {"name": name, **c}


def _select(name, *, batch=1, out=8, kv=8, dim=128, dtype="bf16", ctx=32768, room=40000, bf=32, levels=3):
    c = {"kind": "select", "batch": batch, "out": out, "kv": kv, "dim": dim, "dtype": dtype, "ctx": ctx, "room": room, "bf": bf,
         "levels": levels}
    return c if name is None else {"name": name, **c}


def _reorder(name, *, what="tails", batch=8, kv=8, dim=128, dtype="bf16", ctx=100, room=256, bf=32, moved=0.5):
    c = {"kind": "reorder", "what": what, "batch": batch, "kv": kv, "dim": dim, "dtype": dtype, "ctx": ctx, "room": room, "bf": bf,
         "levels": 3, "moved": moved}
    return c if name is None else {"name": name, **c}


def _rotate(name, *, batch=1, length=1, heads=32, kv=8, dim=128, rotary=128, dtype="bf16", table="fp32", interleaved=False,
            norm=True):
    c = {"kind": "rotate", "batch": batch, "length": length, "heads": heads, "kv": kv, "dim": dim, "rotary": rotary, "dtype": dtype,
         "table": table, "interleaved": interleaved, "norm": norm}
    return c if name is None else {"name": name, **c}


def listed():
    return [
        # two answers to one short question, first token of each: latency only
        _attend("attend_n2_ctx300", branches=2, ctx=300, tail=1),
        # sixteen samples of one answer over a document of the single-sequence configuration's length
        _attend("attend_n16_ctx32768", branches=16, ctx=32768, tail=64),
        # the longest context, 64 continuations a few hundred tokens in: 256 query rows a key head
        _attend("attend_n64_ctx131072", branches=64, ctx=131072, tail=256),
        # three padded prompts, five beams each, three drafted tokens checked at once, small heads, an odd group
        _attend("attend_p3_n5_d64_lq3_ragged", prompts=3, branches=5, kv=4, group=3, dim=64, ctx=9001, tail=37, lq=3, ragged=True),
        # full precision, ragged
        _attend("attend_p2_n4_fp32", prompts=2, branches=4, group=2, dtype="fp32", ctx=4100, tail=33, ragged=True),
        # an indexed prompt forked into eight sequences, each with room to grow
        _select("select_fork8_ctx32768", batch=1, out=8),
        # finished sequences leave a batch of short ones: full precision, two levels, small heads
        _select("select_12to7_ctx2000_fp32", batch=12, out=7, kv=4, dim=64, dtype="fp32", ctx=2000, room=2500, bf=16, levels=2),
        # a quarter of the sequences of a batch replaced by copies of others, indexes of 16,384 tokens
        _reorder("reorder_index_b8_ctx16384", what="index", batch=8, ctx=16384, room=20000, moved=0.25),
        # the tails of eight beams, a hundred tokens in: half of the beams die
        _reorder("reorder_tails_b8_t100", batch=8, ctx=100, room=256, moved=0.5),
        # one token of one sequence: latency only
        _rotate("rotate_b1_l1"),
        # one step of a batch of branches; tables in the model's type, no norms
        _rotate("rotate_b64_l1", batch=64, table="bf16", norm=False),
        # a prompt, partly rotated heads
        _rotate("rotate_l8191_r64", length=8191, rotary=64),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "select", "reorder", "rotate", "rotate"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    kv = rng.choice([1, 2, 4, 8, 8])
    dim = rng.choice([64, 128, 128, 128, 96])
    if kind == "attend":
        group = rng.choice([1, 2, 3, 4, 4, 5, 8])
        lq = rng.choice([1, 1, 1, 1, 2, 5])
        prompts = rng.choice([1, 1, 1, 2, 3])
        branches = _log_int(rng, 1, 64)
        rows = prompts * branches * kv * group * lq
        # no more than a quarter of the largest listed case's products; full precision runs them more slowly
        most = 64 * 8 * 4 * 131072 // (4 if dtype == "bf16" else 64) // rows
        ctx = _log_int(rng, 1, max(2, min(131072 // prompts, most)))
        return _attend(None, prompts=prompts, branches=branches, kv=kv, group=group, dim=dim, dtype=dtype, ctx=ctx,
                       tail=_log_int(rng, lq, 700), lq=lq, ragged=rng.choice([False, True]))
    if kind == "select":
        batch = rng.choice([1, 1, 2, 5, 12])
        out = rng.randint(1, 8 if batch < 5 else batch)
        ctx = _log_int(rng, 200, 32768 // max(batch, out) * 2)
        return _select(None, batch=batch, out=out, kv=kv, dim=dim, dtype=dtype, ctx=ctx, room=ctx + rng.randint(0, ctx // 2),
                       bf=rng.choice([16, 32, 32, 64]), levels=rng.choice([2, 3, 3]))
    if kind == "reorder":
        what = rng.choice(["tails", "tails", "index"])
        batch = rng.randint(2, 48 if what == "tails" else 8)
        ctx = _log_int(rng, 1, 1000) if what == "tails" else _log_int(rng, 200, 16384)
        return _reorder(None, what=what, batch=batch, kv=kv, dim=dim, dtype=dtype, ctx=ctx, room=ctx + rng.randint(0, ctx),
                        bf=rng.choice([16, 32]), moved=rng.choice([0.1, 0.25, 0.5, 0.9]))
    length = rng.choice([1, 1, _log_int(rng, 2, 16384)])
    batch = _log_int(rng, 1, 256) if length == 1 else rng.choice([1, 2])
    return _rotate(None, batch=batch, length=length // batch if length > 1 else 1, heads=kv * rng.choice([1, 3, 4, 8]), kv=kv, dim=dim,
                   rotary=rng.choice([dim, dim, dim // 2, 24]), dtype=dtype, table=rng.choice(["fp32", dtype]),
                   interleaved=rng.choice([False, False, True]), norm=rng.choice([True, False]))


# ---- attend -----------------------------------------------------------------------------------------
def _lens(case):
    """Keys each prompt and each branch's tail really hold."""
    p, n, ctx, tail = case["prompts"], case["branches"], case["ctx"], case["tail"]
    if not case["ragged"]:
        return [ctx] * p, [tail] * (p * n)
    return ([max(1, ctx - (ctx * i) // (2 * p)) for i in range(p)],
            [max(case["lq"], tail - (5 * b) % max(1, tail)) for b in range(p * n)])


def _prepare_attend(case, g):
    p, n, kv, d, ctx, tail, lq = (case[x] for x in ("prompts", "branches", "kv", "dim", "ctx", "tail", "lq"))
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda")
    # keys with a few loud channels, as cached keys have them; queries that make some keys stand out
    loud = torch.ones(d, device="cuda")
    loud[[3, d // 4, d // 2 + 1, d - 2]] = 3.0
    s = {"q": (randn(p * n, lq, kv * case["group"], d) * 1.25).to(dt).transpose(1, 2),
         "pk": (randn(p, kv, ctx, d) * loud).to(dt), "pv": randn(p, kv, ctx, d).to(dt),
         "tk": (randn(p * n, kv, tail, d) * loud).to(dt), "tv": randn(p * n, kv, tail, d).to(dt), "plens": None, "tlens": None}
    if case["ragged"]:
        pl, tl = _lens(case)
        s["plens"] = torch.tensor(pl, dtype=torch.int32, device="cuda")
        s["tlens"] = torch.tensor(tl, dtype=torch.int32, device="cuda")
    return s


def _run_attend(case, s):
    q, pk, pv, tk, tv = s["q"], s["pk"], s["pv"], s["tk"], s["tv"]
    if own:
        from hira_b200 import hira_shared_attention
        return hira_shared_attention(q, pk, pv, tk, tv, prefix_lens=s["plens"], tail_lens=s["tlens"])
    p, n, kv, grp, lq = (case[x] for x in ("prompts", "branches", "kv", "group", "lq"))
    d, ctx, tail = case["dim"], case["ctx"], case["tail"]
    x = q.float().reshape(p, n, kv, grp * lq, d) * d ** -0.5
    s_pre = x.transpose(1, 2).reshape(p, kv, n * grp * lq, d) @ pk.float().transpose(-1, -2)      # (p, kv, rows, ctx)
    s_tail = x.reshape(p * n, kv, grp * lq, d) @ tk.float().transpose(-1, -2)                     # (b, kv, grp * lq, tail)
    at = torch.arange(tail, device="cuda")
    tlens = torch.full((p * n,), tail, device="cuda") if s["tlens"] is None else s["tlens"]
    seen = tlens[:, None] - (lq - 1 - torch.arange(lq, device="cuda"))[None, :]                   # (b, lq) tail keys in sight
    hidden = (at[None, None, :] >= seen[:, :, None])[:, None, None].expand(-1, kv, grp, -1, -1).reshape(s_tail.shape)
    s_tail = s_tail.masked_fill(hidden, float("-inf"))
    if s["plens"] is not None:
        gone = torch.arange(ctx, device="cuda")[None, :] >= s["plens"][:, None]
        s_pre = s_pre.masked_fill(gone[:, None, None, :], float("-inf"))
    s_tail = s_tail.reshape(p, n, kv, grp * lq, tail).transpose(1, 2).reshape(p, kv, n * grp * lq, tail)
    m = torch.maximum(s_pre.amax(-1, keepdim=True), s_tail.amax(-1, keepdim=True))
    e_pre, e_tail = torch.exp(s_pre - m), torch.exp(s_tail - m)
    total = e_pre.sum(-1, keepdim=True) + e_tail.sum(-1, keepdim=True)
    o = e_pre @ pv.float()
    e_tail = e_tail.reshape(p, kv, n, grp * lq, tail).transpose(1, 2).reshape(p * n, kv, grp * lq, tail)
    o_tail = (e_tail @ tv.float()).reshape(p, n, kv, grp * lq, d).transpose(1, 2).reshape(o.shape)
    o = ((o + o_tail) / total).reshape(p, kv, n, grp, lq, d)
    return o.permute(0, 2, 1, 3, 4, 5).reshape(p * n, kv * grp, lq, d).to(q.dtype)


def _exact_attend(case, s):
    p, n, kv, grp, lq, d = (case[x] for x in ("prompts", "branches", "kv", "group", "lq", "dim"))
    pl, tl = _lens(case)
    q = s["q"].double()
    out = torch.zeros((p * n, kv * grp, lq, d), dtype=torch.float64, device="cuda")
    for i in range(p):
        for h in range(kv):
            heads = slice(h * grp, (h + 1) * grp)
            keys, vals = s["pk"][i, h, :pl[i]].double(), s["pv"][i, h, :pl[i]].double()
            scores = torch.einsum("bgtd,kd->bgtk", q[i * n:(i + 1) * n, heads], keys) / math.sqrt(d)
            for j in range(n):
                b = i * n + j
                ext = torch.einsum("gtd,kd->gtk", q[b, heads], s["tk"][b, h, :tl[b]].double()) / math.sqrt(d)
                for t in range(lq):
                    ext[:, t, max(0, tl[b] - (lq - 1 - t)):] = float("-inf")
                w = torch.softmax(torch.cat([scores[j], ext], dim=-1), dim=-1)
                out[b, heads] = torch.einsum("gtk,kd->gtd", w, torch.cat([vals, s["tv"][b, h, :tl[b]].double()]))
    return out


def _work_attend(case):
    p, n, kv, grp, lq, d = (case[x] for x in ("prompts", "branches", "kv", "group", "lq", "dim"))
    e = 2 if case["dtype"] == "bf16" else 4
    pl, tl = _lens(case)
    pairs = sum(x * n * lq for x in pl) + sum(max(0, x - t) for x in tl for t in range(lq))
    return {"bytes": e * d * kv * (2 * sum(pl) + 2 * sum(tl) + 2 * p * n * grp * lq), "flops": 4 * d * kv * grp * pairs}


# ---- select, reorder --------------------------------------------------------------------------------
def _shape(case):
    """(parents in use, grandparents in use, parents there is room for, grandparents there is room for) of each head."""
    bf, three = case["bf"], case["levels"] == 3
    parents, cap = -(-case["ctx"] // bf), -(-case["room"] // bf)
    if not three:
        return parents, 0, cap, 0
    g, cap_g = -(-parents // bf), -(-cap // bf)
    return g * bf, g, cap_g * bf, cap_g


def _index(case, g):
    """The arrays of a built index, heads folded with the sequences; what is not in use is empty."""
    h, d, bf, dt = case["batch"] * case["kv"], case["dim"], case["bf"], DTYPES[case["dtype"]]
    p, gp, cap_p, cap_g = _shape(case)

    def part(cap, used, *tail, dtype=dt, empty=0):
        t = torch.full((h, cap, *tail), empty, dtype=dtype, device="cuda")
        x = torch.randn((h, used, *tail), generator=g, device="cuda")
        t[:, :used] = x.to(dtype) if dtype.is_floating_point else (x * 1000).abs().to(dtype)
        return t
    a = {"children": part(cap_p * bf, p * bf, d), "values": part(cap_p * bf, p * bf, d),
         "slot2token": part(cap_p * bf, p * bf, dtype=torch.int32, empty=-1),
         "parents": part(cap_p, p, d), "parent_radii": part(cap_p, p, dtype=torch.float32),
         "parent_sqnorm": part(cap_p, p, dtype=torch.float32), "child_counts": part(cap_p, p, dtype=torch.int32)}
    if case["levels"] == 3:
        a.update({"grand_parents": part(cap_g, gp, d), "gp_radii": part(cap_g, gp, dtype=torch.float32),
                  "gp_sqnorm": part(cap_g, gp, dtype=torch.float32), "gp_counts": part(cap_g, gp, dtype=torch.int32)})
    a["used"] = torch.tensor([p, gp, case["ctx"], 0], dtype=torch.int32, device="cuda").repeat(h, 1)
    return a


def _picks(case, g):
    b = case["batch"]
    if case["kind"] == "select":
        if case["out"] >= b:                        # every sequence forked, the first ones once more than the others
            return (torch.arange(case["out"], device="cuda") * b // case["out"]).long()
        return torch.randperm(b, generator=g, device="cuda")[:case["out"]].sort().values     # some leave, the rest close up
    # some sequences die and are replaced by copies of survivors, which stay where they are
    dead = torch.randperm(b, generator=g, device="cuda")[:max(1, min(b - 1, round(case["moved"] * b)))]
    alive = torch.ones(b, dtype=torch.bool, device="cuda").index_fill_(0, dead, False).nonzero().flatten()
    idx = torch.arange(b, device="cuda")
    idx[dead] = alive[torch.randint(len(alive), (len(dead),), generator=g, device="cuda")]
    return idx


def _prepare_gather(case, g):
    s = {"idx": _picks(case, g)}
    if case["kind"] == "reorder" and case["what"] == "tails":
        shape = (case["batch"], case["kv"], case["ctx"], case["dim"])
        k, v = (torch.randn(shape, generator=g, device="cuda").to(DTYPES[case["dtype"]]) for _ in range(2))
        if not own:
            s.update(k=k, v=v)
            return s
        from hira_b200 import SharedPrompt
        prefix = torch.zeros((1, case["kv"], 1, case["dim"]), dtype=k.dtype, device="cuda")
        s["prompt"] = SharedPrompt(prefix, prefix, case["batch"], max_tail=case["room"])
        s["prompt"].append(k, v)
        return s
    arrays = _index(case, g)
    if not own:
        s["arrays"] = arrays
        return s
    from hira_b200 import CUDAIndexer
    p, gp, cap_p, _ = _shape(case)
    names = {"bf16": "torch.bfloat16", "fp32": "torch.float32"}
    meta = dict(n_heads=case["batch"] * case["kv"], dim=case["dim"], vdim=case["dim"], bf=case["bf"], depth=case["levels"],
                cap_parents=cap_p, dtype=names[case["dtype"]], vdtype=names[case["dtype"]], n_keys=case["ctx"],
                parents_bound=p, gp_bound=gp, batch=case["batch"])
    s["indexer"] = CUDAIndexer.from_state_dict({**arrays, "meta": meta})
    return s


def _run_gather(case, s):
    idx, b = s["idx"], case["batch"]
    if own and "prompt" in s:
        s["prompt"].reorder(idx)
        return [s["prompt"].tail_keys, s["prompt"].tail_values]
    if own:
        if case["kind"] == "select":
            arrays = s["indexer"].select(idx).state_dict()
        else:
            s["indexer"].reorder(idx)
            arrays = s["indexer"].state_dict()
        return [arrays[name] for name in sorted(arrays) if name != "meta"]
    if "arrays" not in s:
        for t in (s["k"], s["v"]):
            t.copy_(t[idx])
        return [s["k"], s["v"]]
    out = []
    for name in sorted(s["arrays"]):
        a = s["arrays"][name]
        new = a.view(b, case["kv"], *a.shape[1:])[idx].flatten(0, 1)
        out.append(new if case["kind"] == "select" else a.copy_(new))
    return out


def _work_gather(case):
    e, d, kv = (2 if case["dtype"] == "bf16" else 4), case["dim"], case["kv"]
    if case["kind"] == "reorder" and case["what"] == "tails":
        rows = 2 * kv * case["ctx"] * d * e
    else:
        p, gp, _, _ = _shape(case)
        rows = kv * (p * case["bf"] * (2 * d * e + 4) + p * (d * e + 12) + gp * (d * e + 12) + 16)
    if case["kind"] == "select":
        read, written = min(case["batch"], case["out"]), case["out"]
    else:
        written = max(1, min(case["batch"] - 1, round(case["moved"] * case["batch"])))
        read = min(written, case["batch"] - written)
    return {"bytes": (read + written) * rows, "flops": 0}


# ---- rotate -----------------------------------------------------------------------------------------
def _prepare_rotate(case, g):
    b, n, d, r, dt = case["batch"], case["length"], case["dim"], case["rotary"], DTYPES[case["dtype"]]

    def heads(h):      # as a projection leaves them: token by token, all heads of a token together
        x = torch.randn((b, n, h, d), generator=g, device="cuda") * (0.5 + torch.rand((b, n, h, 1), generator=g, device="cuda"))
        return x.to(dt).transpose(1, 2)
    first = torch.randint(0, 131072 - n, (b, 1), generator=g, device="cuda")
    pos = (first + torch.arange(n, device="cuda")).double()
    freq = ROPE_BASE ** (-torch.arange(0, r, 2, device="cuda", dtype=torch.float64) / r)
    angle = pos[:, :, None] * freq
    angle = angle.repeat_interleave(2, -1) if case["interleaved"] else torch.cat([angle, angle], -1)
    s = {"q": heads(case["heads"]), "k": heads(case["kv"]), "cos": angle.cos().to(DTYPES[case["table"]]),
         "sin": angle.sin().to(DTYPES[case["table"]]), "qw": None, "kw": None}
    if case["norm"]:
        s["qw"], s["kw"] = ((1 + 0.3 * torch.randn(d, generator=g, device="cuda")).to(dt) for _ in range(2))
    return s


def _run_rotate(case, s):
    if own:
        from hira_b200 import hira_qk_norm_rope
        return hira_qk_norm_rope(s["q"], s["k"], s["cos"], s["sin"], q_weight=s["qw"], k_weight=s["kw"], eps=EPS,
                                 interleaved=case["interleaved"])
    r, half = case["rotary"], case["rotary"] // 2
    cos, sin = s["cos"].float()[:, None], s["sin"].float()[:, None]
    out = []
    for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])):
        y = x.float()
        if w is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * w.float()
        turn = y[..., :r]
        if case["interleaved"]:
            other = torch.stack([-turn[..., 1::2], turn[..., 0::2]], dim=-1).flatten(-2)
        else:
            other = torch.cat([-turn[..., half:], turn[..., :half]], dim=-1)
        out.append(torch.cat([turn * cos + other * sin, y[..., r:]], dim=-1).to(x.dtype))
    return out


def _exact_rotate(case, s):
    r, half = case["rotary"], case["rotary"] // 2
    first = torch.arange(0, r, 2, device="cuda") if case["interleaved"] else torch.arange(half, device="cuda")
    second = first + (1 if case["interleaved"] else half)
    cos, sin = s["cos"].double().unsqueeze(1), s["sin"].double().unsqueeze(1)
    out = []
    for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])):
        x = x.double()
        if w is not None:
            x = w.double() * x / torch.sqrt(x.square().sum(-1, keepdim=True) / case["dim"] + EPS)
        y = x.clone()
        y[..., first] = x[..., first] * cos[..., first] - x[..., second] * sin[..., first]
        y[..., second] = x[..., second] * cos[..., second] + x[..., first] * sin[..., second]
        out.append(y)
    return out


def _work_rotate(case):
    e, tokens = (2 if case["dtype"] == "bf16" else 4), case["batch"] * case["length"]
    values = tokens * (case["heads"] + case["kv"]) * case["dim"]
    table = 2 * tokens * case["rotary"] * (2 if case["table"] == "bf16" else 4)
    return {"bytes": 2 * e * values + table + (2 * e * case["dim"] if case["norm"] else 0), "flops": values * (7 if case["norm"] else 3)}


# ---- the four of them -------------------------------------------------------------------------------
_PREPARE = {"attend": _prepare_attend, "select": _prepare_gather, "reorder": _prepare_gather, "rotate": _prepare_rotate}
_RUN = {"attend": _run_attend, "select": _run_gather, "reorder": _run_gather, "rotate": _run_rotate}
_WORK = {"attend": _work_attend, "select": _work_gather, "reorder": _work_gather, "rotate": _work_rotate}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return {"case": case, **_PREPARE[case["kind"]](case, g)}


@torch.no_grad()
def run(state):
    return _RUN[state["case"]["kind"]](state["case"], state)


def work(case):
    return _WORK[case["kind"]](case)


@torch.no_grad()
def exact(case, seed):
    """64-bit results of what is computed; copies have none."""
    if case["kind"] not in ("attend", "rotate"):
        return None
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    if case["kind"] == "attend":
        return _exact_attend(case, _prepare_attend(case, g))
    return _exact_rotate(case, _prepare_rotate(case, g))
