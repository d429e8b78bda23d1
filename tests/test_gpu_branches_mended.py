"""Several continuations of one prompt: calls that once went wrong, and the ones beside them."""
import pytest
import torch
from transformers import LlamaConfig

from hira_b200 import (CacheOutput, CUDAIndexer, HiraCache, HiraCacheLayer, HiraConfig, SharedPrompt, hira_attention, hira_qk_norm_rope,
                       hira_shared_attention, patch_attention)
from hira_b200 import _lib as L
from hira_b200 import index_state as S
from test_patched_layers_host import D, HIDDEN, _Layer, _neighbours

pytestmark = pytest.mark.gpu


def _cache_of_one_layer():
    layer = HiraCacheLayer("cuda_only", 4, dict(num_levels=2, max_iterations=1, branching_factor=8), {})

    class One:
        def update(self, k, v, idx):
            return layer.update(k, v)
    return One()


@torch.no_grad()
@pytest.mark.parametrize("rotary", [D, 8])
@pytest.mark.parametrize("odd", ["", "table_halves"])
def test_interleaved_layers_rotate_as_their_own_forward_does(odd, rotary):
    """Tables by channel, and tables that hold a pair's value at i and i + R/2."""
    layer = _Layer(odd, pairs=_neighbours, rotary=rotary).cuda()
    model = torch.nn.ModuleList([layer])
    model.register_buffer("inv_freq", torch.ones(rotary // 2))
    n, gen = 20, torch.Generator().manual_seed(5)
    x = (torch.randn((1, n, HIDDEN), generator=gen) * 20).cuda()
    angle = torch.randn((1, n, rotary // 2), generator=gen).cuda() * 6
    angle = torch.cat([angle, angle], -1) if odd else angle.repeat_interleave(2, -1)
    mask = torch.full((1, 1, n, n), torch.finfo(torch.float32).min, device="cuda").triu(1)
    want = layer(x, (angle.cos(), angle.sin()), mask)[0]
    assert patch_attention(model, interleaved=True) == 1
    got = layer(x, position_embeddings=(angle.cos(), angle.sin()), past_key_values=_cache_of_one_layer())[0]
    torch.testing.assert_close(got, want, atol=1e-4, rtol=1e-3)


@pytest.mark.parametrize("depth", [2, 3])
def test_a_fork_of_an_index_without_its_int8_copy_finds_the_keys_appended_since(depth):
    """The appends do not keep up a copy that is switched off, so a fork must not search by it."""
    gen = torch.Generator().manual_seed(1)
    k, v = (torch.randn((2, 2, 600, 128), generator=gen).bfloat16().cuda() for _ in range(2))
    ix = CUDAIndexer(depth, 1, 16, max_context=626).build(k, v)
    assert ix.state.cap_parents % 64 == 0        # whole tiles, which the search by the copy needs
    ix.state.enable_int8_copy(False)
    new = k[:, :, :4] * 3
    ix.update(new, v[:, :, :4])
    q = torch.nn.functional.normalize(new.float(), dim=-1)           # four queries a head, each along a new key
    tau = torch.full((16,), 15.0, device="cuda")
    flags = L.HIRA_GATE_GE | L.HIRA_LEAF_GE
    picks = [1, 0]
    fork = ix.select(picks)
    got = S.search(fork.state, q[picks].reshape(16, 128), tau, flags=flags, want_compact=True)[1].to_lists()
    want = S.search(ix.state, q.reshape(16, 128), tau, flags=flags, want_compact=True)[1].to_lists()
    for i in range(16):
        j = picks[i // 8] * 8 + i % 8
        assert len(want[j][0]) > 0 and torch.equal(got[i][0], want[j][0]) and torch.equal(got[i][1], want[j][1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_lengths_beyond_32_bits_are_cut_like_others(dtype):
    gen = torch.Generator().manual_seed(2)
    q, pk, pv, tk, tv = (torch.randn(s, generator=gen).to(dtype).cuda()
                         for s in ((4, 2, 1, 64), (2, 1, 90, 64), (2, 1, 90, 64), (4, 1, 9, 64), (4, 1, 9, 64)))
    want = hira_shared_attention(q, pk, pv, tk, tv, prefix_lens=[90, 0], tail_lens=[9, 9, 0, 3])
    far = torch.tensor([2 ** 32 + 5, -2 ** 32 + 5, 2 ** 31, -2 ** 31 - 1], device="cuda")
    got = hira_shared_attention(q, pk, pv, tk, tv, prefix_lens=far[:2], tail_lens=torch.stack([far[0], far[2], far[3], far.new_tensor(3)]))
    assert torch.equal(got, want)
    prompt = SharedPrompt(pk, pv, 2, prefix_lens=far[:2]).append(tk, tv)
    assert torch.equal(prompt.attend(q), hira_shared_attention(q, pk, pv, tk, tv, prefix_lens=[90, 0]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_heads_of_one_projection_rotate_in_place_and_into_each_other(dtype):
    """Views that lie between each other share no byte; calls of one layout with outputs at other places."""
    gen = torch.Generator().manual_seed(3)
    b, n, d = 2, 5, 64
    qw, kw = (torch.randn(d, generator=gen).to(dtype).cuda() for _ in range(2))
    angle = torch.randn((b, n, d), generator=gen).cuda()
    cos, sin = angle.cos(), angle.sin()
    for _ in range(3):
        fused = torch.randn((b, n, 12, d), generator=gen).to(dtype).cuda().transpose(1, 2)
        q, k, old = fused[:, :4], fused[:, 4:6], fused.clone()
        want = hira_qk_norm_rope(q.clone(), k.clone(), cos, sin, q_weight=qw, k_weight=kw)
        hira_qk_norm_rope(q, k, cos, sin, q_weight=qw, k_weight=kw, out_q=fused[:, 6:10], out_k=fused[:, 10:])
        assert torch.equal(fused[:, :6], old[:, :6]) and torch.equal(fused[:, 6:10], want[0]) and torch.equal(fused[:, 10:], want[1])
        hira_qk_norm_rope(q, k, cos, sin, q_weight=qw, k_weight=kw, out_q=q, out_k=k)
        assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(fused[:, 6:10], want[0])
        with pytest.raises(ValueError, match="apart"):        # the layout of the first call, at another place
            hira_qk_norm_rope(q, k, cos, sin, q_weight=qw, k_weight=kw, out_q=fused[:, 5:9], out_k=fused[:, 10:])
        with pytest.raises(ValueError, match="same memory"):
            hira_qk_norm_rope(q, k, cos, sin, q_weight=qw, k_weight=kw, out_q=fused[:, 6:10], out_k=fused[:, 8:10])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("ctx,tail,group,branches", [(300, 7, 2, 3), (40, 9, 5, 20), (6000, 300, 1, 4), (0, 5, 4, 2), (33, 0, 4, 40)])
def test_attention_over_its_own_query_and_between_others(dtype, ctx, tail, group, branches):
    gen = torch.Generator().manual_seed(4)
    h, d = 2, 64
    kv = [torch.randn(s, generator=gen).to(dtype).cuda() for s in ((1, h, ctx, d), (1, h, ctx, d), (branches, h, tail, d), (branches, h, tail, d))]
    for _ in range(3):
        fused = torch.randn((branches, 2 * h * group + 3, 1, d), generator=gen).to(dtype).cuda()
        q, other, old = fused[:, :h * group], fused[:, h * group:2 * h * group], fused.clone()
        want = hira_shared_attention(q.clone(), *kv)
        assert hira_shared_attention(q, *kv, out=other) is other
        assert torch.equal(other, want) and torch.equal(q, old[:, :h * group]) and torch.equal(fused[:, 2 * h * group:], old[:, 2 * h * group:])
        with pytest.raises(ValueError, match="query"):
            hira_shared_attention(q, *kv, out=fused[:, 1:1 + h * group])
        hira_shared_attention(q, *kv, out=q)
        assert torch.equal(q, want) and torch.equal(other, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("queued", [0, 3])
def test_a_prompt_shared_on_another_stream_is_whole_although_the_index_is_dropped(queued, dtype):
    gen = torch.Generator().manual_seed(6)
    k, v = (torch.randn((2, 2, 3000 + queued, 128), generator=gen).to(dtype).cuda() for _ in range(2))
    layer = HiraCacheLayer("cuda_only", 8, dict(num_levels=3, max_iterations=1, branching_factor=16), {})
    layer.update(k[:, :, :3000], v[:, :, :3000])
    if queued:
        layer.update(k[:, :, 3000:], v[:, :, 3000:])
    slow = torch.randn((4096, 4096), device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(40):                          # keeps what follows on the side stream waiting
            slow = torch.nn.functional.normalize(slow @ slow)
        layer.share_prompt(3)
    # takes freed memory of the first stream, if any is
    junk = [torch.full(s, 7.0, dtype=d, device="cuda") for s, d in
            [((4, 4096, 128), dtype)] * 6 + [((2, 2, 8, 128), dtype)] * 6 + [((4, 4096), torch.float32)] * 6]
    torch.cuda.synchronize()
    del junk
    assert torch.equal(layer.shared.prefix_keys, k) and torch.equal(layer.shared.prefix_values, v)
    assert layer.get_seq_length() == 3000 + queued


@pytest.mark.parametrize("tail", [0, 4])
def test_a_bad_index_is_still_reported_after_forks_and_without_a_tail(tail):
    k = torch.randn((1, 2, 9, 16), device="cuda")

    def prompt():
        p = SharedPrompt(k, k, 4)
        return p.append(*[torch.randn((4, 2, tail, 16), device="cuda")] * 2) if tail else p
    good, bad = torch.tensor([3, 2, 1, 0], device="cuda"), torch.tensor([0, 1, 2, 4], device="cuda")
    p = prompt().reorder(good).select(good).select([1, 0, 1])
    p.check_status()
    for f in (lambda: prompt().reorder(bad), lambda: prompt().select(bad), lambda: prompt().reorder(bad).select([0, 1]),
              lambda: prompt().reorder(bad).reorder(good).select(good).select([1]), lambda: prompt().select(bad[3:] - 9)):
        with pytest.raises(RuntimeError, match="does not exist"):
            f().check_status()
    layer = HiraCacheLayer("cuda_only", 4, dict(num_levels=2, max_iterations=1, branching_factor=8), {})
    layer.update(k.repeat(2, 1, 8, 1).bfloat16(), k.repeat(2, 1, 8, 1).bfloat16())
    layer.share_prompt(1)
    layer.batch_repeat_interleave(2)
    layer.shared.check_status()


def test_a_bad_index_of_a_captured_reordering_is_reported_without_a_tail():
    k = torch.randn((1, 2, 9, 16), device="cuda")
    p, idx = SharedPrompt(k, k, 4, max_tail=8), torch.arange(4, device="cuda")
    p.reorder(idx)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        p.reorder(idx)
    g.replay()
    p.check_status()
    idx[2] = -1
    g.replay()
    with pytest.raises(RuntimeError, match="does not exist"):
        p.check_status()


def test_what_an_index_has_to_report_is_reported_by_its_shared_prompt():
    k = torch.randn((2, 2, 40, 16), device="cuda").bfloat16()
    for bad in (False, True):
        layer = HiraCacheLayer("cuda_only", 4, dict(num_levels=2, max_iterations=1, branching_factor=8), {})
        layer.update(k, k)
        layer.reorder_cache(torch.tensor([0, 2 if bad else 1], device="cuda"))
        layer.share_prompt(2)
        layer.batch_select_indices([0, 2])
        if bad:
            with pytest.raises(RuntimeError, match="does not exist"):
                layer.shared.check_status()
        else:
            layer.shared.check_status()


def test_a_cache_shares_the_prompts_of_all_its_layers_or_of_none():
    cfg = LlamaConfig(vocab_size=8, hidden_size=32, num_hidden_layers=3, num_attention_heads=2, num_key_value_heads=2, head_dim=16)
    cache = HiraCache(cfg, HiraConfig(device_mode="cuda_only", update_every=4, num_levels=2, branching_factor=8))
    k = torch.randn((2, 2, 40, 16), device="cuda")

    def unchanged(match, **kw):
        with pytest.raises(ValueError, match=match):
            cache.share_prompt(**{**dict(branches=2), **kw})
        assert all(layer.shared is None for layer in cache.layers)
    cache.update(k, k, 0)
    cache.update(k, k, 1)
    unchanged("no prompt")
    cache.update(k, k.bfloat16(), 2)
    unchanged("one type")
    cache.layers[2].reset()
    cache.update(k, k, 2)
    unchanged("branches", branches=0)
    cache.share_prompt(2)
    assert all(layer.shared.batch == 4 for layer in cache.layers)
    with pytest.raises(ValueError, match="already"):
        cache.share_prompt(2)


def test_attention_leaves_what_its_status_holds():
    gen = torch.Generator().manual_seed(7)
    k, v, q = (torch.randn(s, generator=gen).bfloat16().cuda() for s in ((1, 2, 40000, 128), (1, 2, 40000, 128), (9, 8, 1, 128)))
    for word in (0, 2):
        status = torch.full((1,), word, dtype=torch.int32, device="cuda")
        out = hira_shared_attention(q, k, v, status=status)
        assert torch.isfinite(out).all() and int(status) == word and torch.equal(out, hira_shared_attention(q, k, v))
    prompt = SharedPrompt(k, v, 9)
    prompt.attend(q)
    prompt.check_status()


def _counted(p, n, h, g, lq, d, v, ctx, tail, dtype, plens=None, tlens=None):
    """Every key counts: with queries of 0 all weights are 1, so an output is a number of keys over a number of keys.  Each channel
    has 1 at 64 keys in turn, so that one key too few or too many moves it by 1/64, four times the rounding of bf16; as many
    calls as it takes to have every key in some channel."""
    b = p * n
    gen = torch.Generator().manual_seed(8)
    q = torch.zeros((b, h * g, lq, d), dtype=dtype, device="cuda")
    pk, tk = (torch.randn(s, generator=gen).to(dtype).cuda() for s in ((p, h, ctx, d), (b, h, tail, d)))
    pl = torch.full((p,), ctx, device="cuda") if plens is None else torch.tensor(plens, device="cuda")
    tl = torch.full((b,), tail, device="cuda") if tlens is None else torch.tensor(tlens, device="cuda")
    owner = torch.arange(b, device="cuda") // n
    seen_t = (tl[:, None] - (lq - 1 - torch.arange(lq, device="cuda"))[None]).clamp(min=0)        # (b, lq)
    total = (pl[owner][:, None] + seen_t).double()
    half = 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -8
    chan = torch.arange(v, device="cuda")
    for turn in range(-(-max(ctx, tail) // (64 * v))):
        first = (chan + turn * v) * 64                                  # channel c has 1 at keys first[c] .. first[c] + 63

        def values(rows):
            at = torch.arange(rows, device="cuda")
            return ((at[:, None] >= first[None]) & (at[:, None] < first[None] + 64)).to(dtype)

        def among(length):                                              # of the first `length` keys
            return (length[..., None] - first).clamp(0, 64)
        pv, tv = values(ctx).expand(p, h, ctx, v).contiguous(), values(tail).expand(b, h, tail, v).contiguous()
        want = (among(pl[owner])[:, None] + among(seen_t)).double() / total[..., None].clamp(min=1)
        got = hira_shared_attention(q, pk, pv, tk, tv, prefix_lens=None if plens is None else pl, tail_lens=None if tlens is None else tl)
        # the quotient as a reciprocal and a product in 32 bits (2^-23), then the rounding
        off = (got.double() - want[:, None]).abs() - want[:, None] * (half + 2.0 ** -22)
        assert (off <= 0).all(), f"turn {turn}: off by {off.max().item():.3g} more than a rounding"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [
    # p, n, h, g, lq, d, v, ctx, tail
    (1, 8, 1, 1, 1, 128, 128, 131072, 0),         # one key head: many splits
    (1, 8, 1, 1, 1, 128, 128, 131072, 1),         # joined by the tails' blocks
    (1, 4, 1, 2, 1, 64, 64, 400000, 3),
    (1, 3, 2, 4, 1, 128, 128, 65536, 700),
    (1, 16, 2, 4, 1, 64, 64, 40000, 130),
    (1, 16, 8, 4, 1, 128, 128, 20000, 64),        # 64 rows a key head, tiles dealt out in runs
    (2, 33, 3, 4, 1, 128, 128, 9001, 130),        # 132 rows
    (3, 5, 4, 3, 3, 64, 64, 9001, 37),
    (1, 70, 1, 8, 1, 64, 64, 20001, 2),           # 560 rows
    (1, 4, 1, 2, 1, 256, 256, 70000, 33),
    (2, 20, 2, 4, 1, 256, 256, 3001, 129),
    (1, 5, 1, 3, 2, 136, 64, 20000, 260),
    (1, 2, 1, 1, 1, 128, 128, 0, 70000),          # a long tail alone
    (1, 2, 1, 2, 1, 128, 128, 70001, 70001),      # both long
], ids=lambda s: "x".join(map(str, s)))
def test_every_key_counts(shape, dtype):
    _counted(*shape, dtype)
    p, n, _, _, _, _, _, ctx, tail = shape
    _counted(*shape, dtype, plens=[ctx - 77 * i if i else max(0, ctx - 1) for i in range(p)], tlens=[max(0, tail - 3 * i) for i in range(p * n)])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("share", [True, False])
def test_a_captured_step_of_a_cache_reorders_appends_and_attends(share, dtype):
    """A step of a search over continuations, captured once over a cache of two layers and replayed with other picks and tokens, does
    what the same calls do one by one (the tail's length is the host's: each replay writes the same row)."""
    cfg = LlamaConfig(vocab_size=8, hidden_size=128, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=64)
    gen = torch.Generator().manual_seed(9)

    def rnd(*shape):
        return torch.randn(shape, generator=gen).to(dtype).cuda()
    prompts = [(rnd(1, 2, 230, 64), rnd(1, 2, 230, 64)) for _ in range(2)]
    queued = [(rnd(1, 2, 3, 64), rnd(1, 2, 3, 64)) for _ in range(2)]           # not yet indexed
    tokens = [(rnd(6, 2, 5, 64), rnd(6, 2, 5, 64)) for _ in range(2)]

    def cache():
        c = HiraCache(cfg, HiraConfig(device_mode="cuda_only", update_every=64, num_levels=2, branching_factor=8, max_context=400,
                                      threshold_method="none"))
        for i in range(2):
            c.update(*prompts[i], i)
            c.update(*queued[i], i)
        c.share_prompt(6, max_tail=16) if share else c.batch_repeat_interleave(6)
        for i in range(2):
            c.update(*tokens[i], i)
        return c

    def step(c, picks, q, new):
        c.reorder_cache(picks)
        outs = []
        for i in range(2):
            out, _ = c.update(*new[i], i)
            outs.append(hira_attention(None, q, out, None, None, scaling=0.2, hira_config=c.hira_config)[0])
        return outs

    def other_values():
        return torch.randint(6, (6,), generator=gen).cuda(), rnd(6, 4, 1, 64), [(rnd(6, 2, 1, 64), rnd(6, 2, 1, 64)) for _ in range(2)]
    c = cache()
    picks, q, new = other_values()
    if not share:                  # the search's workspaces come into being
        for i in range(2):
            out = c.layers[i]
            hira_attention(None, q, CacheOutput(out.queued_keys, out.queued_values, None, None, out.indexer, out.searcher), None, None,
                           scaling=0.2, hira_config=c.hira_config)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step(c, picks, q, new)
    state = cache()                # goes the same way without a graph
    for _ in range(4):
        values = other_values()
        for static, now in zip([picks, q, *new[0], *new[1]], [values[0], values[1], *values[2][0], *values[2][1]]):
            static.copy_(now)
        g.replay()
        want = step(state, *values)
        for a, b in zip(outs, want):
            assert torch.equal(a, b)
        for a, b in zip(c.layers, state.layers):
            assert torch.equal(a.queued_keys, b.queued_keys) and torch.equal(a.queued_values, b.queued_values)
        for layer in state.layers:             # back to the length that the graph was captured with
            if share:
                layer.shared._len -= 1
            else:
                layer.queued_len -= 1
    for layer in c.layers:
        (layer.shared if share else layer.indexer).check_status()


@pytest.mark.parametrize("shape", [
    # p, n, h, g, d, v, ctx, tail
    (1, 2, 2, 4, 128, 128, 300, 9),               # few rows: 16 rows a block
    (1, 16, 8, 4, 128, 128, 4000, 64),            # 64 rows a key head: two chains over the same rows
    (1, 40, 8, 4, 128, 128, 4000, 70),            # 160 rows: a chain for each 128
    (2, 20, 8, 4, 64, 64, 5000, 3),
    (2, 40, 8, 4, 64, 64, 5000, 3),
    (1, 4, 2, 2, 256, 256, 900, 70),
    (1, 3, 1, 2, 128, 128, 0, 700),               # tails alone
], ids=lambda s: "x".join(map(str, s)))
def test_softmax_weights_are_not_rounded_to_bf16(shape):
    """Logits of one product each, exact in 32 bits, so that what is left is the weights' precision: 2^-15 of each in two terms."""
    p, n, h, g, d, v, ctx, tail = shape
    gen = torch.Generator().manual_seed(10)

    def rnd(*s):
        return torch.randn(s, generator=gen).bfloat16().cuda()
    b = p * n
    q = torch.zeros((b, h * g, 1, d), dtype=torch.bfloat16, device="cuda")
    q[..., 0] = rnd(b, h * g, 1)
    pk, tk = (torch.zeros(s, dtype=torch.bfloat16, device="cuda") for s in ((p, h, ctx, d), (b, h, tail, d)))
    pk[..., 0], tk[..., 0] = rnd(p, h, ctx), rnd(b, h, tail)
    pv, tv = rnd(p, h, ctx, v), rnd(b, h, tail, v)
    scaling = 0.75
    got = hira_shared_attention(q, pk, pv, tk, tv, scaling=scaling)
    for s in range(b):
        for hh in range(h):
            k, w = (torch.cat([x[s // n, hh], y[s, hh]]).double() for x, y in ((pk, tk), (pv, tv)))
            x = q[s, hh * g:(hh + 1) * g, 0].double()
            z = scaling * (x @ k.T)
            probs = torch.softmax(z, dim=-1)
            want, mean = probs @ w, probs @ w.abs()
            # a logit: times the scale and log2(e), less the maximum (2^-24 each of up to 2 x 1.45 |z|), the exponential (2^-22); both in
            # numerator and denominator.  Sums over the keys in 32 bits, cut where the tensor cores add.  The weights.  The output's rounding
            off = 2 * (3 * 2.0 ** -24 * 2 * 1.45 * z.abs().amax(-1, keepdim=True) + 2.0 ** -22) + 2.0 ** -23 * (64 + len(k) / 8) + 2.0 ** -15
            diff = (got[s, hh * g:(hh + 1) * g, 0].double() - want).abs() - (off * mean + 2.0 ** -8 * want.abs())
            assert (diff <= 0).all(), f"off by {diff.max().item():.3g} more than the bound"
