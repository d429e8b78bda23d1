"""Several continuations of one prompt: shared attention, sequences forked / reordered / compacted, norms with rotation.

Every operator against a plain implementation in 64 bits, at the sizes, masks and layouts where it can go wrong."""
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch

from hira_b200 import (CUDAIndexer, HiraCache, HiraConfig, SharedPrompt, hira_attention, hira_decode_attention, hira_qk_norm_rope,
                       hira_shared_attention, patch_attention)
from hira_b200 import index_state as S

pytestmark = pytest.mark.gpu
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}      # half a step, relative to the value


# ---- shared attention ------------------------------------------------------------------------------
def _qkv(p, n, h, g, lq, d, v, ctx, tail, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)

    def r(*shape):
        return torch.randn(shape, generator=gen).to(dtype).cuda()
    return r(p * n, h * g, lq, d), r(p, h, ctx, d), r(p, h, ctx, v), r(p * n, h, tail, d), r(p * n, h, tail, v)


def _exact(q, pk, pv, tk, tv, plens=None, tlens=None, scaling=None):
    """(output in 64 bits, bound on what the kernels may be off by): see `_check`."""
    b, hq, lq, d = q.shape
    p, h, ctx, v = pv.shape
    n, g = b // p, hq // h
    scaling = d ** -0.5 if scaling is None else scaling
    out = torch.zeros((b, hq, lq, v), dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for s in range(b):
        a = s // n
        pl = ctx if plens is None else max(0, min(ctx, int(plens[a])))
        tl = 0 if tk is None else (tk.shape[2] if tlens is None else max(0, min(tk.shape[2], int(tlens[s]))))
        for t in range(lq):
            see = max(0, tl - (lq - 1 - t))
            for hh in range(h):
                k, w = pk[a, hh, :pl], pv[a, hh, :pl]
                if see:
                    k, w = torch.cat([k, tk[s, hh, :see]]), torch.cat([w, tv[s, hh, :see]])
                if len(k) == 0:
                    continue
                k, w, x = k.double(), w.double(), q[s, hh * g:(hh + 1) * g, t].double()
                probs = torch.softmax(scaling * (x @ k.T), dim=-1)
                o, mean = probs @ w, probs @ w.abs()
                # a logit: d products summed in 32 bits (2^-22 a step where the tensor cores cut instead of rounding), times
                # the scale and log2(e), less the maximum, and the exponential itself (2^-22); numerator and denominator
                logit = abs(scaling) * (x.abs() @ k.abs().T).amax(-1, keepdim=True)
                off = 2 * (logit * (d + 8) * 2.0 ** -22 + 2.0 ** -21)
                # sums over the keys in 32 bits; with bf16 each weight is rounded once more; the output once
                off = off + 2.0 ** -23 * (64 + len(k) / 32) + (HALF[q.dtype] if q.dtype == torch.bfloat16 else 0)
                out[s, hh * g:(hh + 1) * g, t] = o
                tol[s, hh * g:(hh + 1) * g, t] = off * mean + HALF[q.dtype] * o.abs() + 1e-30
    return out, tol


def _check(got, want):
    out, tol = want
    off = (got.double() - out).abs() - tol
    assert torch.isfinite(got).all() and (off <= 0).all(), f"off by {off.max().item():.3g} more than the bound"


SHAPES = [
    # p, n, h, g, lq, d, v, ctx, tail
    (1, 1, 1, 1, 1, 128, 128, 1, 1),
    (1, 2, 2, 4, 1, 128, 128, 300, 1),
    (1, 3, 1, 1, 1, 128, 128, 127, 5),
    (1, 1, 2, 1, 1, 64, 64, 128, 64),
    (1, 5, 2, 3, 1, 64, 64, 129, 65),
    (2, 3, 2, 4, 3, 128, 128, 513, 37),
    (3, 2, 1, 8, 2, 96, 96, 200, 17),
    (1, 40, 2, 4, 1, 128, 128, 1000, 3),          # 160 rows a key head: two row tiles
    (1, 70, 1, 8, 1, 64, 64, 400, 2),             # 560 rows: several row blocks
    (2, 33, 3, 4, 1, 128, 128, 4097, 130),
    (1, 4, 2, 2, 1, 8, 8, 77, 9),
    (1, 4, 2, 2, 1, 24, 40, 77, 9),
    (1, 3, 2, 2, 2, 256, 256, 150, 70),
    (1, 3, 2, 2, 1, 128, 256, 150, 70),
    (1, 3, 2, 2, 1, 200, 72, 150, 70),
    (1, 2, 8, 4, 1, 128, 128, 20000, 700),        # many splits of prefix and tail
    (1, 9, 1, 2, 40, 128, 128, 260, 90),          # long drafts: 80 rows a tail
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_shared_attention_equals_attention_of_each_sequence(shape, dtype):
    t = _qkv(*shape, dtype, seed=sum(shape))
    _check(hira_shared_attention(*t), _exact(*t))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128, 160])
def test_lengths_cut_prefix_and_tail_and_what_lies_behind_is_not_used(dtype, d):
    p, n, h, g, lq, ctx, tail = 5, 6, 2, 2, 2, 390, 70
    q, pk, pv, tk, tv = _qkv(p, n, h, g, lq, d, d, ctx, tail, dtype, seed=3)
    plens = [0, 1, 128, 257, 390]
    tlens = [(7 * i) % (tail + 1) for i in range(p * n)]      # 0 among them: rows of an empty prefix that see nothing
    tlens[:6] = [0, 1, 2, 64, 65, 70]
    for a, ln in enumerate(plens):
        pk[a, :, ln:], pv[a, :, ln:] = float("nan"), float("inf")
    for s, ln in enumerate(tlens):
        tk[s, :, ln:], tv[s, :, ln:] = float("-inf"), float("nan")
    want = _exact(q, pk, pv, tk, tv, plens, tlens)
    got = hira_shared_attention(q, pk, pv, tk, tv, prefix_lens=torch.tensor(plens, device="cuda"), tail_lens=torch.tensor(tlens, device="cuda"))
    _check(got, want)
    assert (got[0] == 0).all() and (got[1, :, 0] == 0).all()       # no key in sight
    assert torch.equal(got, hira_shared_attention(q, pk, pv, tk, tv, prefix_lens=plens, tail_lens=tlens))
    beyond = torch.tensor(tlens, device="cuda")                       # on the device lengths are cut to what there is
    beyond[5], beyond[0] = 1000, -4
    assert torch.equal(got, hira_shared_attention(q, pk, pv, tk, tv, prefix_lens=plens, tail_lens=beyond))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prefix_alone_tail_alone_and_nothing(dtype):
    q, pk, pv, tk, tv = _qkv(2, 3, 2, 2, 2, 128, 128, 140, 9, dtype, seed=4)
    _check(hira_shared_attention(q, pk, pv), _exact(q, pk, pv, None, None))
    _check(hira_shared_attention(q, pk[:, :, :0], pv[:, :, :0], tk, tv), _exact(q, pk[:, :, :0], pv[:, :, :0], tk, tv))
    assert (hira_shared_attention(q, pk[:, :, :0], pv[:, :, :0]) == 0).all()
    assert (hira_shared_attention(q, pk[:, :, :0], pv[:, :, :0], tk[:, :, :0], tv[:, :, :0]) == 0).all()
    assert hira_shared_attention(q[:, :, :0], pk, pv, tk, tv).shape == (6, 4, 0, 128)
    assert hira_shared_attention(q[:0], pk, pv).shape == (0, 4, 2, 128)
    # fewer tail keys than query tokens: the first tokens see none of it
    _check(hira_shared_attention(q, pk, pv, tk[:, :, :1], tv[:, :, :1]), _exact(q, pk, pv, tk[:, :, :1], tv[:, :, :1]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts_strides_and_out(dtype):
    p, n, h, g, lq, d, ctx, tail = 2, 3, 2, 2, 2, 64, 200, 21
    q, pk, pv, tk, tv = _qkv(p, n, h, g, lq, d, d, ctx, tail, dtype, seed=5)
    want = _exact(q, pk, pv, tk, tv)
    base = hira_shared_attention(q, pk, pv, tk, tv)
    _check(base, want)

    def tokens_first(t):             # (B, L, H, D) memory, as projections leave it
        return t.transpose(1, 2).contiguous().transpose(1, 2)

    def roomy(t):                    # the filled part of a buffer
        buf = torch.full((*t.shape[:2], t.shape[2] + 13, t.shape[3]), float("nan"), dtype=t.dtype, device="cuda")
        buf[:, :, :t.shape[2]] = t
        return buf[:, :, :t.shape[2]]

    def odd(t):                      # rows that start between 16-byte boundaries: copied
        buf = torch.empty((*t.shape[:3], t.shape[3] + 1), dtype=t.dtype, device="cuda")
        buf[..., 1:] = t
        return buf[..., 1:]

    def strided(t):                  # elements not one behind another: copied
        return t.repeat_interleave(2, dim=-1)[..., ::2]
    for f in (tokens_first, roomy, odd, strided):
        assert torch.equal(base, hira_shared_attention(f(q), f(pk), f(pv), f(tk), f(tv)))
    same = pk[:1].expand(p, -1, -1, -1), pv[:1].expand(p, -1, -1, -1)
    _check(hira_shared_attention(q, *same, tk, tv), _exact(q, same[0].contiguous(), same[1].contiguous(), tk, tv))
    out = torch.full((p * n, lq, h * g, d), float("nan"), dtype=dtype, device="cuda")
    assert hira_shared_attention(q, pk, pv, tk, tv, out=out.transpose(1, 2)).data_ptr() == out.data_ptr()
    assert torch.equal(out.transpose(1, 2), base)
    _check(hira_shared_attention(q, pk, pv, tk, tv, scaling=0.7), _exact(q, pk, pv, tk, tv, scaling=0.7))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scaling", [-0.11, 0.0, 1e-4])
def test_scalings_of_any_sign(dtype, scaling):
    t = _qkv(1, 3, 2, 2, 2, 128, 128, 333, 70, dtype, seed=21)
    _check(hira_shared_attention(*t, scaling=scaling), _exact(*t, scaling=scaling))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_that_overlap_and_tails_of_one_for_all(dtype):
    gen = torch.Generator().manual_seed(22)
    line = torch.randn(8 * 300 + 128, generator=gen).to(dtype).cuda()
    keys = line.as_strided((1, 2, 200, 64), (0, 8 * 50, 8, 1))             # windows of one line
    q, _, pv, tk, tv = _qkv(1, 4, 2, 2, 1, 64, 64, 200, 9, dtype, seed=22)
    tk, tv = tk[:1].expand(4, -1, -1, -1), tv[:1].expand(4, -1, -1, -1)
    _check(hira_shared_attention(q, keys, pv, tk, tv), _exact(q, keys.contiguous(), pv, tk.contiguous(), tv.contiguous()))


def test_tails_of_every_length_through_one_layout():
    """Calls of one layout with a tail that grows, a buffer of one row and one of many, and an `out` of the caller's."""
    q, pk, pv, tk, tv = _qkv(1, 3, 2, 2, 1, 128, 128, 200, 130, torch.bfloat16, seed=23)
    for cap in (1, 2, 130):
        bk, bv = tk[:, :, :cap].contiguous(), tv[:, :, :cap].contiguous()
        for n in [x for x in (0, 1, 2, 3, 63, 64, 65, 128, 130) if x <= cap]:
            want = _exact(q, pk, pv, bk[:, :, :n] if n else None, bv[:, :, :n] if n else None)
            _check(hira_shared_attention(q, pk, pv, bk[:, :, :n], bv[:, :, :n]), want)
            out = torch.full((3, 1, 4, 128), float("nan"), dtype=torch.bfloat16, device="cuda")
            for _ in range(2):
                hira_shared_attention(q, pk, pv, bk[:, :, :n], bv[:, :, :n], out=out.transpose(1, 2))
            _check(out.transpose(1, 2), want)


def test_many_calls_at_once_on_two_streams():
    cases = [(_qkv(2, 5, 2, 4, 1, 128, 128, 700 + 13 * i, 33 + i, torch.bfloat16, seed=30 + i)) for i in range(6)]
    want = [hira_shared_attention(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for rounds in range(5):
        for i, c in enumerate(cases):
            with torch.cuda.stream(streams[i % 2]):
                got.append((i, hira_shared_attention(*c)))
    torch.cuda.synchronize()
    assert all(bool((x == want[i]).all()) for i, x in got)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(2, 20, 2, 4, 1, 256, 256, 1501, 33), (1, 5, 1, 3, 2, 136, 64, 4000, 260), (1, 17, 2, 1, 1, 64, 248, 65, 1),
                                   (1, 1, 40, 4, 1, 256, 256, 700, 16)], ids=lambda s: "x".join(map(str, s)))
def test_wide_rows_in_several_row_blocks_and_splits(shape, dtype):
    q, pk, pv, tk, tv = _qkv(*shape, dtype, seed=81)
    p, b, lens = shape[0], shape[0] * shape[1], [shape[7] - 40] + [0] * (shape[0] - 1)
    _check(hira_shared_attention(q, pk, pv, tk, tv), _exact(q, pk, pv, tk, tv))
    tl = [i % (shape[8] + 1) for i in range(b)]
    pk[:, :, shape[7] - 40:], pv[:, :, shape[7] - 40:] = float("nan"), float("nan")      # behind the lengths
    if p > 1:
        pk[1:], pv[1:] = float("nan"), float("nan")
    _check(hira_shared_attention(q, pk, pv, tk, tv, prefix_lens=lens, tail_lens=tl), _exact(q, pk, pv, tk, tv, lens, tl))


def test_threads_that_call_at_once_with_rows_of_different_widths():
    cases = [_qkv(1, 3, 2, 2, 1, d, v, 150, 70, dtype, seed=50 + d + v)
             for d, v in ((256, 256), (64, 64), (8, 8), (128, 128), (128, 256)) for dtype in (torch.float32, torch.bfloat16)]
    torch.cuda.synchronize()

    def call(c):
        with torch.cuda.stream(torch.cuda.Stream()):
            out = hira_shared_attention(*c)
            torch.cuda.current_stream().synchronize()
        return out
    with ThreadPoolExecutor(len(cases)) as pool:
        got = [list(pool.map(call, cases)) for _ in range(5)]
    for outs in got:
        for c, out in zip(cases, outs):
            _check(out, _exact(*c))


def test_a_scaling_held_in_a_tensor_is_read_at_each_call():
    q, pk, pv, tk, tv = _qkv(1, 3, 2, 2, 1, 64, 64, 100, 5, torch.bfloat16, seed=71)
    scaling = torch.tensor(0.125)
    for value in (0.125, 0.5):
        scaling.fill_(value)
        _check(hira_shared_attention(q, pk, pv, tk, tv, scaling=scaling), _exact(q, pk, pv, tk, tv, scaling=value))
    x, c, s = q[:, :2].float(), torch.ones((1, 64), device="cuda"), torch.zeros((1, 64), device="cuda")
    eps, w = torch.tensor(1e-6), torch.ones(64, device="cuda")
    small = hira_qk_norm_rope(x, x, c, s, q_weight=w, eps=eps)[0]
    eps.fill_(3.0)
    assert torch.equal(hira_qk_norm_rope(x, x, c, s, q_weight=w, eps=eps)[0], hira_qk_norm_rope(x, x, c, s, q_weight=w, eps=3.0)[0])
    assert not torch.equal(small, hira_qk_norm_rope(x, x, c, s, q_weight=w, eps=eps)[0])


def test_large_logits_of_either_sign():
    for dtype in (torch.float32, torch.bfloat16):
        q, pk, pv, tk, tv = _qkv(1, 3, 1, 2, 1, 128, 128, 700, 40, dtype, seed=6)
        for f in (30.0, -30.0):
            got = hira_shared_attention(q * f, pk, pv, tk, tv)
            _check(got, _exact(q * f, pk, pv, tk, tv))
        # rising logits: the running maximum moves on in nearly every tile
        up = torch.linspace(-20, 20, 700, device="cuda").view(1, 1, 700, 1)
        pk2 = (torch.nn.functional.normalize(q[:1, :1].float(), dim=-1) * up).to(dtype)
        _check(hira_shared_attention(q, pk2, pv, tk, tv), _exact(q, pk2, pv, tk, tv))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_nan_in_sight_reaches_the_rows_that_see_it_and_no_other(dtype):
    for where in ("query", "prefix", "tail"):
        q, pk, pv, tk, tv = _qkv(2, 3, 2, 2, 1, 128, 128, 300, 40, dtype, seed=12)
        good = hira_shared_attention(q, pk, pv, tk, tv)
        hit = torch.zeros(6, 4, dtype=torch.bool, device="cuda")
        if where == "query":
            q[4, 1, 0, 5], hit[4, 1] = float("nan"), True
        elif where == "prefix":
            pk[1, 0, 200, 3], hit[3:, :2] = float("nan"), True
        else:
            tk[2, 1, 39, 3], hit[2, 2:] = float("nan"), True
        got = hira_shared_attention(q, pk, pv, tk, tv)
        assert bool(torch.isnan(got[hit]).all()) and bool((got[~hit] == good[~hit]).all()), where
    q, pk, pv, tk, tv = _qkv(1, 2, 1, 2, 1, 64, 64, 300, 40, dtype, seed=13)
    assert bool(torch.isnan(hira_shared_attention(q, pk * float("nan"), pv)).all())


def _in_long_buffer(q, *rows):
    """The prompts' rows at the front of buffers so long (and NaN behind them) that their tiles go to the tcgen05 kernel, which few
    rows and keys do not; and how many of them there are."""
    p, h, n, _ = rows[0].shape
    blocks = -(-q.shape[0] // p * (q.shape[1] // h) * q.shape[2] // 16)
    room = max(n, 1280 * 148 // (blocks * p * h) + 1)
    out = []
    for t in rows:
        buf = torch.full((p, h, room, t.shape[3]), float("nan"), dtype=t.dtype, device="cuda")
        buf[:, :, :n] = t
        out.append(buf)
    return (*out, [n] * p)


@pytest.mark.parametrize("shape", [s for s in SHAPES if max(s[5], s[6]) <= 128], ids=lambda s: "x".join(map(str, s)))
def test_short_prompts_in_long_buffers(shape):
    q, pk, pv, tk, tv = _qkv(*shape, torch.bfloat16, seed=91)
    bk, bv, lens = _in_long_buffer(q, pk, pv)
    _check(hira_shared_attention(q, bk, bv, tk, tv, prefix_lens=lens), _exact(q, pk, pv, tk, tv))
    _check(hira_shared_attention(q, bk, bv, prefix_lens=lens), _exact(q, pk, pv, None, None))
    for scaling in (-0.11, 0.0):
        _check(hira_shared_attention(q, bk, bv, tk, tv, prefix_lens=lens, scaling=scaling), _exact(q, pk, pv, tk, tv, scaling=scaling))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [2, 17])
def test_lengths_in_long_buffers(n, d):
    p, h, g, lq, tail = 6, 2, 4, 2, 5
    lens = [0, 1, 127, 128, 129, 390]
    q, pk, pv, tk, tv = _qkv(p, n, h, g, lq, d, d, 390, tail, torch.bfloat16, seed=92)
    for a, ln in enumerate(lens):
        pk[a, :, ln:], pv[a, :, ln:] = float("nan"), float("inf")
    bk, bv, _ = _in_long_buffer(q, pk, pv)
    tl = [i % (tail + 1) for i in range(p * n)]
    got = hira_shared_attention(q, bk, bv, tk, tv, prefix_lens=torch.tensor(lens, device="cuda"), tail_lens=tl)
    _check(got, _exact(q, pk, pv, tk, tv, lens, tl))
    assert (got[0] == 0).all()                   # no key in sight
    tokens_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, bk, bv, tk, tv)]
    out = torch.full((p * n, lq, h * g, d), float("nan"), dtype=torch.bfloat16, device="cuda").transpose(1, 2)
    assert torch.equal(hira_shared_attention(*tokens_first, prefix_lens=lens, tail_lens=tl, out=out), got)


def test_logits_and_nans_in_long_buffers():
    q, pk, pv, tk, tv = _qkv(1, 5, 2, 4, 1, 128, 128, 700, 40, torch.bfloat16, seed=93)
    bk, bv, lens = _in_long_buffer(q, pk, pv)
    for f in (30.0, -30.0):
        _check(hira_shared_attention(q * f, bk, bv, tk, tv, prefix_lens=lens), _exact(q * f, pk, pv, tk, tv))
    up = torch.linspace(-20, 20, 700, device="cuda").view(1, 1, 700, 1)      # the running maximum moves on in every tile
    pk2 = (torch.nn.functional.normalize(q[:1, :1].float(), dim=-1) * up).to(torch.bfloat16).expand_as(pk)
    bk2, _, _ = _in_long_buffer(q, pk2, pv)
    _check(hira_shared_attention(q, bk2, bv, tk, tv, prefix_lens=lens), _exact(q, pk2, pv, tk, tv))
    good = hira_shared_attention(q, bk, bv, tk, tv, prefix_lens=lens)
    bk[0, 1, 300, 7] = float("nan")
    got = hira_shared_attention(q, bk, bv, tk, tv, prefix_lens=lens)
    assert torch.equal(got[:, :4], good[:, :4]) and bool(torch.isnan(got[:, 4:]).all())
    bk[0, 1, 300, 7] = 0.0
    static = [x.clone() for x in (q, tk, tv)]
    want = hira_shared_attention(q, bk, bv, tk, tv, prefix_lens=lens)
    dev_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(hira_shared_attention(static[0], bk, bv, *static[1:], prefix_lens=dev_lens))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):                            # two at once
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_prefix_beyond_two_gibi_elements():
    h, d, ctx = 1, 128, (1 << 24) + 77         # 2^31 elements and more: offsets beyond 32 bits
    k = torch.zeros((1, h, ctx, d), dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    q = torch.ones((2, 1, 1, d), dtype=torch.bfloat16, device="cuda")
    k[0, 0, -3:] = 4.0                          # the last keys take all the weight: 4 * 128 / sqrt(128) = 45
    v[0, 0, -3:] = torch.tensor([1.0, 2.0, 6.0], device="cuda")[:, None].bfloat16()
    got = hira_shared_attention(q, k, v)
    assert ((got.float() - 3.0).abs() <= 3 * 2.0 ** -8 * 2).all()


def test_captured_replayed_and_on_a_side_stream():
    for dtype, d in ((torch.bfloat16, 128), (torch.float32, 64)):
        t = _qkv(2, 4, 2, 2, 1, d, d, 600, 33, dtype, seed=7)
        want = hira_shared_attention(*t)
        t2 = _qkv(2, 4, 2, 2, 1, d, d, 600, 33, dtype, seed=8)
        want2 = hira_shared_attention(*t2)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            a, b = hira_shared_attention(*t), hira_shared_attention(*t2)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(a, want) and torch.equal(b, want2)
        static = [x.clone() for x in t]
        g1, g2, g3 = (torch.cuda.CUDAGraph() for _ in range(3))
        with torch.cuda.graph(g1):
            o1 = hira_shared_attention(*static)
        with torch.cuda.graph(g2):
            o2 = hira_shared_attention(*static)
        with torch.cuda.graph(g3, pool=g2.pool()):      # graphs that share a pool replay in the order of their capture
            o3 = hira_shared_attention(*static)
        g1.replay()
        assert bool((o1 == want).all())
        for x, y in zip(static, t2):
            x.copy_(y)
        g2.replay()
        g3.replay()
        g1.replay()
        torch.cuda.synchronize()
        for o in (o1, o2, o3):
            assert bool((o == want2).all())


# ---- sequences forked, reordered, compacted --------------------------------------------------------------
PICKS = [[0], [0, 0, 0], [1, 0], [2, 0, 1], [0, 1, 2, 3], [3, 3, 1, 0], [1, 2, 3, 4, 0, 0, 0], [5, 4, 3, 2, 1, 0], [2, 2, 2, 5, 5, 5]]


@pytest.mark.parametrize("rows,dim,dtype", [(1, 8, torch.float32), (37, 64, torch.bfloat16), (513, 128, torch.bfloat16), (70, 1, torch.float32)])
@pytest.mark.parametrize("picks", PICKS, ids=str)
def test_rows_gathered_into_other_memory_and_in_place(picks, rows, dim, dtype):
    n, h, cap, used = max(len(picks), max(picks) + 1), 3, rows + 5, rows
    gen = torch.Generator().manual_seed(rows)
    src = torch.randn((n, h, cap, dim), generator=gen).to(dtype).cuda()
    idx = torch.tensor(picks, device="cuda")
    dst = torch.full((len(picks), h, cap, dim), 7.0, dtype=dtype, device="cuda")
    S.gather_rows(S.RowMoves([(src, dst)]), idx, used)
    assert torch.equal(dst[:, :, :used], src[idx][:, :, :used]) and (dst[:, :, used:] == 7).all()
    full = torch.cat([idx, torch.arange(len(picks), n, device="cuda")])
    want = src.clone()
    want[:, :, :used] = src[full][:, :, :used]
    S.gather_rows(S.RowMoves([(src, src)]), full, used)
    assert torch.equal(src, want)


@pytest.mark.parametrize("n", [2, 8, 12, 17, 32, 100, 769, 2048])
def test_many_sequences_permuted_in_place(n):
    gen = torch.Generator().manual_seed(n)
    src = torch.randn((n, 2, 9, 8), generator=gen).cuda()
    for idx in (torch.randperm(n, generator=gen), torch.randint(n, (n,), generator=gen), torch.roll(torch.arange(n), 1)):
        want = src[idx.cuda()].clone()
        S.gather_rows(S.RowMoves([(src, src)]), idx.cuda(), 9)
        assert torch.equal(src, want)


def test_a_sequence_that_does_not_exist_changes_nothing_and_is_reported():
    src = torch.randn((4, 2, 8, 16), device="cuda")
    keep, status = src.clone(), torch.zeros(1, dtype=torch.int32, device="cuda")
    S.gather_rows(S.RowMoves([(src, src)]), torch.tensor([1, 4, -1, 0], device="cuda"), 8, status)
    assert torch.equal(src, keep[[1, 1, 2, 0]]) and int(status) == 8
    prompt = SharedPrompt(keep[:1], keep[:1], 4, max_tail=8).append(keep, keep)
    prompt.check_status()
    prompt.reorder(torch.tensor([0, 1, 2, 9], device="cuda"))
    with pytest.raises(RuntimeError, match="does not exist"):
        prompt.check_status()
    ix = _index(2, 2, 300, 64, torch.bfloat16, 3)[0]
    before = {k: v.clone() for k, v in ix.state_dict().items() if k != "meta"}
    ix.reorder(torch.tensor([0, 2], device="cuda"))
    assert all(torch.equal(before[k], v) for k, v in ix.state_dict().items() if k != "meta")
    with pytest.raises(RuntimeError, match="does not exist"):
        ix.check_status()


def _index(b, h, n, d, dtype, depth, bf=16, max_context=None, seed=0):
    gen = torch.Generator().manual_seed(seed)
    k = torch.randn((b, h, n, d), generator=gen).to(dtype).cuda()
    v = torch.randn((b, h, n, d), generator=gen).to(dtype).cuda()
    ix = CUDAIndexer(depth, 1, bf, max_context=max_context)
    ix.build(k, v)
    return ix, k, v


def _arrays(ix):
    names = [n for n in S.IndexState.ARRAYS + S.IndexState.Q8_ARRAYS if getattr(ix.state, n) is not None and n != "q8_query_scratch"]
    a = {n: getattr(ix.state, n).view(ix.batch, -1, *getattr(ix.state, n).shape[1:]) for n in names}
    for n in ("children_q8", "children_q8_meta"):         # of free slots nothing is kept there
        if n in a:
            free = a["slot2token"] < 0
            a[n] = a[n].masked_fill(free if a[n].ndim == 3 else free[..., None], 0)
    return a


@pytest.mark.parametrize("depth", [2, 3])
@pytest.mark.parametrize("dtype,d,n,room", [(torch.bfloat16, 128, 1000, 1500), (torch.float32, 64, 333, None), (torch.bfloat16, 96, 50, 400)])
def test_selected_index_holds_the_picked_sequences(depth, dtype, d, n, room):
    ix, k, v = _index(4, 2, n, d, dtype, depth, max_context=room)
    ix.update(k[:, :, :3] * 0.5, v[:, :, :3])
    old = {a: t.clone() for a, t in _arrays(ix).items()}
    for picks in ([0], [3, 1], [0, 0, 1, 1, 2, 2, 3, 3], [2, 3, 0, 1]):
        new = ix.select(picks)
        got = _arrays(new)
        for a in old:
            assert torch.equal(got[a], old[a][picks]), a
        assert new.batch == len(picks) and new.num_heads == 2 * len(picks)
        # what the picked sequences do afterwards is what they would have done: append, search, attend
        alone = _index(1, 2, n, d, dtype, depth, max_context=room)[0]
        for j, b in enumerate(picks[:2]):
            one = CUDAIndexer.from_state_dict({**{a: t[b] for a, t in old.items() if a in S.IndexState.ARRAYS},
                                               "meta": {**ix.state_dict()["meta"], "n_heads": 2, "batch": 1}})
            del alone
            alone = one
            step_k, step_v = k[b:b + 1, :, 5:6] * 1.1, v[b:b + 1, :, 7:8]
            alone.update(step_k, step_v)
            fork = ix.select(picks).update(k[picks, :, 5:6] * 1.1, v[picks, :, 7:8])
            for a in S.IndexState.ARRAYS:
                t = getattr(fork.state, a)
                if t is not None:
                    assert torch.equal(t.view(len(picks), 2, *t.shape[1:])[j], getattr(alone.state, a)), a
    for a, t in _arrays(ix).items():
        assert torch.equal(t, old[a])


@pytest.mark.parametrize("depth", [2, 3])
@pytest.mark.parametrize("picks", [[0, 1, 2], [2, 0, 1], [1, 1, 1], [0, 2, 2]])
def test_reordered_index_attends_as_its_new_sequences(depth, picks):
    from hira_b200 import CUDASearcher, CacheOutput
    d = 128
    ix, k, v = _index(3, 2, 700, d, torch.bfloat16, depth, max_context=900)
    q = torch.randn((3, 4, 1, d), device="cuda")

    def attend(index, query, **kw):
        return hira_decode_attention(query, CacheOutput(None, None, None, None, index, CUDASearcher()), scaling=0.2, sample_size=64, topk=8, **kw)
    before = attend(ix, q[[picks.index(b) if b in picks else 0 for b in range(3)]])      # draws the samples of the threshold
    old = {a: t.clone() for a, t in _arrays(ix).items()}
    ix.begin_scanned_update(k[:, :, :1])
    ix.reorder(torch.tensor(picks, device="cuda"))
    for a, t in _arrays(ix).items():
        assert torch.equal(t, old[a][picks]), a
    got = attend(ix, q)
    for j, b in enumerate(picks):
        if picks.index(b) == j:
            assert torch.equal(got[j], before[b])       # the threshold's samples have moved with their sequences
    with pytest.raises(ValueError, match="scanned"):
        ix.update(k[:, :, :1], v[:, :, :1], scanned=True)
    ix.update(k[:, :, :1], v[:, :, :1])
    ix.check_status()


def test_every_set_of_samples_follows_its_sequences():
    from hira_b200.attention.hira_attention import _samples_for
    ix, k, v = _index(4, 2, 500, 64, torch.bfloat16, 3)
    sets = [_samples_for(ix, s) for s in (32, 64, 100)]
    before = [s.clone() for s in sets]
    ix.reorder([3, 0, 0, 1])
    for s, old in zip(sets, before):
        assert torch.equal(s.view(4, 2, *s.shape[1:]), old.view(4, 2, *s.shape[1:])[[3, 0, 0, 1]])


def test_an_update_on_a_side_stream_waits_for_the_reordering():
    from hira_b200 import CUDASearcher, CacheOutput
    ix, k, v = _index(3, 2, 2000, 128, torch.bfloat16, 3, max_context=3000)
    ref = ix.select([0, 1, 2])         # (the channel scales of the int8 copy differ between two builds)
    q, side = torch.randn((3, 4, 1, 128), device="cuda"), torch.cuda.Stream()
    for t in range(4):
        picks = torch.tensor([(t + 1) % 3, t % 3, 0], device="cuda")
        for index, stream in ((ix, side), (ref, None)):
            hira_decode_attention(q, CacheOutput(None, None, None, None, index, CUDASearcher()), threshold_method="none")
            index.reorder(picks)
            index.update(k[:, :, t:t + 1] * 0.9, v[:, :, t:t + 1], stream=stream)
    ix.wait_pending_update()
    torch.cuda.synchronize()
    for a, t in _arrays(ix).items():
        assert torch.equal(t, _arrays(ref)[a]), a


def test_an_index_selected_on_another_stream_is_whole_when_the_old_one_is_dropped():
    ix, k, v = _index(2, 2, 20000, 128, torch.bfloat16, 3)
    want = {a: t[[1, 0, 1]].clone() for a, t in _arrays(ix).items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        new = ix.select([1, 0, 1])
    del ix
    junk = [torch.full((1 << 26,), 7, dtype=torch.int32, device="cuda") for _ in range(4)]      # takes freed memory, if any is
    torch.cuda.synchronize()
    del junk
    for a, t in _arrays(new).items():
        assert torch.equal(t, want[a]), a


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_shared_prompt_follows_its_sequences(dtype):
    p, n, h, g, d = 2, 3, 2, 2, 64
    q, pk, pv, tk, tv = _qkv(p, n, h, g, 1, d, d, 150, 40, dtype, seed=9)
    prompt = SharedPrompt(pk, pv, n)
    for a, b in ((0, 1), (1, 20), (20, 21), (21, 40)):           # grows on the way
        prompt.append(tk[:, :, a:b], tv[:, :, a:b])
    _check(prompt.attend(q), _exact(q, pk, pv, tk, tv))
    idx = torch.tensor([2, 0, 0, 3, 5, 4], device="cuda")
    prompt.reorder(idx)
    tk, tv = tk[idx], tv[idx]
    assert torch.equal(prompt.tail_keys, tk) and torch.equal(prompt.tail_values, tv)
    _check(prompt.attend(q), _exact(q, pk, pv, tk, tv))
    few = prompt.select([2, 0, 3, 4])
    assert few.batch == 4 and torch.equal(few.tail_keys, tk[[2, 0, 3, 4]]) and torch.equal(prompt.tail_keys, tk)
    _check(few.attend(q[:4]), _exact(q[:4], pk, pv, tk[[2, 0, 3, 4]], tv[[2, 0, 3, 4]]))
    with pytest.raises(ValueError, match="apart"):
        prompt.reorder([3, 1, 2, 0, 4, 5])
    with pytest.raises(ValueError, match="apart"):
        prompt.select([0, 1, 2])


# ---- norms with rotation ---------------------------------------------------------------------------------
def _rope_exact(x, cos, sin, w, eps, interleaved):
    """(result in 64 bits, bound): the sum of squares, its root's reciprocal (2 ulp), three products and a sum, in 32 bits."""
    r, d = cos.shape[-1], x.shape[-1]
    y = x.double()
    if w is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * w.double()
    c, s = cos.double()[:, None], sin.double()[:, None]
    first = torch.arange(0, r, 2, device=x.device) if interleaved else torch.arange(r // 2, device=x.device)
    second = first + (1 if interleaved else r // 2)
    out, mag = y.clone(), y.abs()
    out[..., first] = y[..., first] * c[..., first] - y[..., second] * s[..., first]
    out[..., second] = y[..., second] * c[..., second] + y[..., first] * s[..., second]
    mag[..., first] = (y[..., first] * c[..., first]).abs() + (y[..., second] * s[..., first]).abs()
    mag[..., second] = (y[..., second] * c[..., second]).abs() + (y[..., first] * s[..., second]).abs()
    return out, mag * 2.0 ** -24 * (d / 16 + 12) + out.abs() * HALF[x.dtype] + 1e-37


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dtype,table", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16),
                                         (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("b,n,hq,hk,d,r", [(1, 1, 32, 8, 128, 128), (3, 5, 4, 1, 64, 64), (2, 17, 6, 3, 96, 96), (1, 130, 5, 5, 128, 64),
                                           (2, 3, 3, 2, 256, 256), (1, 7, 2, 2, 8, 8), (2, 9, 4, 2, 72, 20), (1, 4, 1, 1, 200, 6), (1, 2, 2, 1, 64, 0)])
def test_norm_and_rotation(b, n, hq, hk, d, r, dtype, table, norm, interleaved):
    gen = torch.Generator().manual_seed(d + r + n)

    def rnd(*shape):
        return torch.randn(shape, generator=gen).cuda()
    q, k = rnd(b, n, hq, d).to(dtype).transpose(1, 2), rnd(b, n, hk, d).to(dtype).transpose(1, 2)
    angle = rnd(b, n, max(r, 1))[..., :r] * 50
    cos, sin = angle.cos().to(table), angle.sin().to(table)      # every channel of its own: the pairs need not agree
    qw, kw = ((1 + 0.3 * rnd(d)).to(dtype) if norm else None for _ in range(2))
    got = hira_qk_norm_rope(q, k, cos, sin, q_weight=qw, k_weight=kw, eps=1e-5, interleaved=interleaved)
    for x, w, y in ((q, qw, got[0]), (k, kw, got[1])):
        out, tol = _rope_exact(x, cos, sin, w, 1e-5, interleaved)
        assert y.shape == x.shape and y.dtype == dtype and ((y.double() - out).abs() <= tol).all()
    # one table for all sequences, in place, and into part of a cache
    if b > 1:
        one = hira_qk_norm_rope(q[:1], k[:1], cos[:1], sin[:1], q_weight=qw, k_weight=kw, eps=1e-5, interleaved=interleaved)
        both = hira_qk_norm_rope(q, k, cos[:1], sin[0], q_weight=qw, k_weight=kw, eps=1e-5, interleaved=interleaved) if r else got
        if r:
            assert torch.equal(both[0][:1], one[0]) and torch.equal(both[1][:1], one[1])
    cache = torch.full((b, hk, n + 7, d), 3.0, dtype=dtype, device="cuda")
    q2, k2 = q.clone(memory_format=torch.preserve_format), k.clone()
    hira_qk_norm_rope(q2, k2, cos, sin, q_weight=qw, k_weight=kw, eps=1e-5, interleaved=interleaved, out_q=q2, out_k=cache[:, :, 2:n + 2])
    assert torch.equal(q2, got[0]) and torch.equal(cache[:, :, 2:n + 2], got[1])
    assert (cache[:, :, :2] == 3).all() and (cache[:, :, n + 2:] == 3).all() and torch.equal(k2, k)


def test_norm_of_zeros_huge_values_and_one_side_only():
    q = torch.zeros((1, 2, 3, 64), device="cuda")
    k = torch.full((1, 1, 3, 64), 1e15, device="cuda")
    cos, sin = torch.ones((1, 3, 64), device="cuda"), torch.zeros((1, 3, 64), device="cuda")
    a, b = hira_qk_norm_rope(q, k, cos, sin, q_weight=torch.ones(64, device="cuda"))
    assert (a == 0).all() and torch.equal(b, k)
    a, b = hira_qk_norm_rope(q, k, cos, sin, k_weight=torch.ones(64, device="cuda"))
    assert torch.equal(a, q) and ((b - 1).abs() <= 2.0 ** -21).all()
    assert hira_qk_norm_rope(q[:, :, :0], k[:, :, :0], cos[:, :0], sin[:, :0])[0].shape == (1, 2, 0, 64)
    f = torch.randn((2, 4, 6 * 64), device="cuda").view(2, 4, 6, 64).transpose(1, 2)      # a fused projection, in place
    want = hira_qk_norm_rope(f[:, :4].clone(), f[:, 4:].clone(), torch.ones((4, 64), device="cuda"), torch.full((4, 64), 0.5, device="cuda"))
    hira_qk_norm_rope(f[:, :4], f[:, 4:], torch.ones((4, 64), device="cuda"), torch.full((4, 64), 0.5, device="cuda"), out_q=f[:, :4], out_k=f[:, 4:])
    assert torch.equal(f[:, :4], want[0]) and torch.equal(f[:, 4:], want[1])


# ---- together, as a model uses them ------------------------------------------------------------------------
def _tiny_llama(**kw):
    from transformers import LlamaConfig, LlamaForCausalLM
    torch.manual_seed(0)
    cfg = LlamaConfig(vocab_size=512, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=64, max_position_embeddings=2048, **kw)
    return cfg, LlamaForCausalLM(cfg).cuda().eval()


@torch.no_grad()
@pytest.mark.parametrize("share", [False, True])
def test_patched_model_continues_a_prompt_many_times_like_dense_attention(share):
    """Prompts, each continued by several sequences that are forked, reordered and dropped on the way."""
    from transformers import DynamicCache
    cfg, model = _tiny_llama()
    _, plain = _tiny_llama()
    hcfg = HiraConfig(device_mode="cuda_only", update_every=3, num_levels=3, branching_factor=8, max_context=500, threshold_method="none")
    assert patch_attention(model, hcfg) == 2
    ids = torch.randint(0, 512, (2, 300), device="cuda")
    cache, ref = HiraCache(cfg, hcfg), DynamicCache(config=cfg)

    def step(tok):
        a = model(tok, past_key_values=cache, use_cache=True).logits
        b = plain(tok, past_key_values=ref, use_cache=True).logits
        torch.testing.assert_close(a, b, atol=2e-3, rtol=2e-3)
        assert cache.get_seq_length(0) == ref.get_seq_length(0)
        return b
    step(ids)
    step(ids[:, 10:11])                                   # one token of the prompt apart: queued, or in the prefix
    cache.share_prompt(3) if share else cache.batch_repeat_interleave(3)
    ref.batch_repeat_interleave(3)
    moves = {1: torch.tensor([1, 1, 0, 5, 4, 3], device="cuda"), 4: torch.tensor([2, 1, 2, 3, 3, 3], device="cuda")}
    for t in range(7):
        logits = step(torch.randint(0, 512, (6, 1), device="cuda"))
        assert logits.shape[0] == 6
        if t in moves:
            cache.reorder_cache(moves[t])
            ref.reorder_cache(moves[t])
    keep = torch.tensor([0, 2, 4, 5], device="cuda")
    cache.batch_select_indices(keep)
    ref.batch_select_indices(keep)
    for _ in range(3):
        step(torch.randint(0, 512, (4, 1), device="cuda"))
    cache.batch_repeat_interleave(2)
    ref.batch_repeat_interleave(2)
    step(torch.randint(0, 512, (8, 1), device="cuda"))
    if share:
        step(torch.randint(0, 512, (8, 3), device="cuda"))           # three drafted tokens at once


class _HeadNorm(torch.nn.Module):
    def __init__(self, width, eps):
        super().__init__()
        self.weight = torch.nn.Parameter(1 + 0.2 * torch.randn(width))
        self.variance_epsilon = eps

    def forward(self, x):
        y = x.float()
        return (y * torch.rsqrt(y.square().mean(-1, keepdim=True) + self.variance_epsilon)).to(x.dtype) * self.weight


@torch.no_grad()
def test_patched_layers_norm_their_heads():
    cfg, model = _tiny_llama()
    layer = model.model.layers[0].self_attn
    layer.q_norm, layer.k_norm = _HeadNorm(64, 1e-5).cuda(), _HeadNorm(64, 1e-5).cuda()
    hcfg = HiraConfig(device_mode="cuda_only", update_every=1, num_levels=2, branching_factor=8, max_context=100, threshold_method="none")
    patch_attention(model, hcfg)
    cache = HiraCache(cfg, hcfg)
    x = torch.randn((1, 20, 256), device="cuda")
    angle = torch.rand((1, 20, 32), device="cuda").repeat(1, 1, 2) * 6
    got, _ = layer(x, position_embeddings=(angle.cos(), angle.sin()), past_key_values=cache)
    q, k, v = (proj(x).view(1, 20, -1, 64).transpose(1, 2).double() for proj in (layer.q_proj, layer.k_proj, layer.v_proj))
    q, k = (_turn(t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-5) * nm.weight.double(), angle.double())
            for t, nm in ((q, layer.q_norm), (k, layer.k_norm)))
    s = q @ k.repeat_interleave(2, dim=1).transpose(-1, -2) / 8
    s = s.masked_fill(torch.triu(torch.ones(20, 20, device="cuda", dtype=torch.bool), 1), float("-inf"))
    want = (torch.softmax(s, -1) @ v.repeat_interleave(2, dim=1)).transpose(1, 2).reshape(1, 20, -1) @ layer.o_proj.weight.double().T
    torch.testing.assert_close(got.double(), want, atol=1e-4, rtol=1e-3)
    layer.k_norm = torch.nn.LayerNorm(64).cuda()
    with pytest.raises(ValueError, match="RMS norm"):
        patch_attention(model, hcfg)


def _turn(x, angle):
    a, b = x[..., :32], x[..., 32:]
    c, s = angle[:, None, :, :32].cos(), angle[:, None, :, :32].sin()
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def test_attention_of_a_shared_layer_goes_through_hira_attention_only():
    q, pk, pv, tk, tv = _qkv(1, 2, 2, 2, 1, 64, 64, 100, 5, torch.bfloat16, seed=11)
    from hira_b200 import HiraCacheLayer
    layer = HiraCacheLayer("cuda_only", 1, dict(num_levels=2, max_iterations=1, branching_factor=8), {})
    with pytest.raises(ValueError, match="no prompt"):
        layer.share_prompt(2)
    layer.update(pk, pv)
    layer.share_prompt(2, max_tail=4)
    with pytest.raises(ValueError, match="already"):
        layer.share_prompt(2)
    out, _ = layer.update(tk, tv)
    assert torch.equal(layer.shared.prefix_keys, pk) and layer.get_seq_length() == 105
    got, _ = hira_attention(None, q, out, None, None)
    _check(got.transpose(1, 2), _exact(q, pk, pv, tk, tv))
    with pytest.raises(ValueError, match="shared"):
        hira_decode_attention(q, out)
    layer.reset()
    layer.update(pk, pv)
    assert layer.shared is None and layer.get_seq_length() == 100
