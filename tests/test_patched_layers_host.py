"""Which attention layers `patch_attention` takes: those whose own forward is what the new one computes, and no others (CPU)."""
import copy
from types import SimpleNamespace

import pytest
import torch

from hira_b200 import patch_attention

HIDDEN, HEADS, KV, D = 48, 4, 2, 16


class _RMS(torch.nn.Module):
    def __init__(self, width, weight=None):
        super().__init__()
        self.weight = torch.nn.Parameter(torch.ones(width) if weight is None else weight)
        self.variance_epsilon = 1e-6

    def forward(self, x):
        y = x.float()
        return self.weight * (y * torch.rsqrt(y.square().mean(-1, keepdim=True) + self.variance_epsilon)).to(x.dtype)


def _halves(x):
    a, b = x.chunk(2, dim=-1)
    return torch.cat([-b, a], dim=-1)


def _neighbours(x):
    return torch.stack([-x[..., 1::2], x[..., 0::2]], dim=-1).flatten(-2)


class _Layer(torch.nn.Module):
    """An attention layer with a forward of its own; `odd` names what it does differently."""

    def __init__(self, odd="", pairs=_halves, rotary=D, head_norms=False, bias=False, scaling=None, kv=KV, dtype=torch.float32, seed=0):
        super().__init__()
        g = torch.Generator().manual_seed(seed)

        def lin(i, o):
            m = torch.nn.Linear(i, o, bias=bias, dtype=dtype)
            for p in m.parameters():
                p.data = (torch.randn(p.shape, generator=g) * 0.02).to(dtype)      # as models are initialised: nearly flat softmax
            return m
        self.layer_idx, self.head_dim, self.odd, self.pairs, self.rotary = 0, D, odd, pairs, rotary
        if scaling is not None:
            self.scaling = scaling
        self.q_proj, self.k_proj, self.v_proj = lin(HIDDEN, HEADS * D * (2 if odd == "gate" else 1)), lin(HIDDEN, kv * D), lin(HIDDEN, kv * D)
        self.o_proj = lin(HEADS * D, HIDDEN)
        self.config = SimpleNamespace()
        if head_norms:
            self.q_norm, self.k_norm = (_RMS(D, 1 + 0.3 * torch.randn(D, generator=g).to(dtype)) for _ in range(2))
        if odd == "sub_norm":
            self.attn_sub_norm = _RMS(HEADS * D)
        if odd == "norm_behind_rotation":
            self.query_layernorm = _RMS(D)
        if odd == "learned_mask":
            self.A = torch.nn.Parameter(torch.zeros(kv))

    def forward(self, hidden_states, position_embeddings, attention_mask=None, past_key_values=None, **kwargs):
        b, n, _ = hidden_states.shape
        q, k, v = (p(hidden_states) for p in (self.q_proj, self.k_proj, self.v_proj))
        if self.odd == "gate":
            q, gate = q.chunk(2, dim=-1)
        if self.odd == "clip":
            q, k, v = (t.clamp(-3, 3) for t in (q, k, v))
        q, k, v = (t.view(b, n, -1, D).transpose(1, 2) for t in (q, k, v))
        if hasattr(self, "q_norm") and self.odd != "norms_unused":
            q, k = self.q_norm(q), self.k_norm(k)
        cos, sin = (t[:, None, :, :self.rotary] for t in position_embeddings)
        if self.odd == "table_halves":
            cos, sin = (t[..., :t.shape[-1] // 2].repeat_interleave(2, dim=-1) for t in (cos, sin))
        r = cos.shape[-1]
        if self.odd != "no_rotation":
            q, k = (torch.cat([t[..., :r] * cos + self.pairs(t[..., :r]) * sin, t[..., r:]], dim=-1) for t in (q, k))
        if self.odd == "norm_behind_rotation":
            q = self.query_layernorm(q)
        if self.odd == "temperature":
            q = q * 1.1
        s = getattr(self, "scaling", D ** -0.5) * (q @ k.repeat_interleave(HEADS // k.shape[1], 1).transpose(-1, -2))
        if self.odd == "cap":
            s = 30.0 * torch.tanh(s / 30.0)
        if attention_mask is not None:
            s = s + attention_mask
        p = torch.softmax(s, dim=-1, dtype=torch.float32).to(s.dtype)
        if self.odd == "sink":
            p = torch.softmax(torch.cat([s, torch.zeros_like(s[..., :1])], -1), -1)[..., :-1]
        if self.odd == "difference":
            p = p - 0.2 * p.roll(1, dims=1)
        o = (p @ v.repeat_interleave(HEADS // v.shape[1], 1)).transpose(1, 2).reshape(b, n, -1)
        if self.odd == "gate":
            o = o * torch.sigmoid(gate)
        if self.odd == "sub_norm":
            o = self.attn_sub_norm(o)
        return self.o_proj(o), None


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("kw", [{}, dict(head_norms=True), dict(bias=True), dict(scaling=0.05), dict(kv=4), dict(kv=1), dict(dtype=torch.bfloat16),
                                dict(head_norms=True, dtype=torch.bfloat16)], ids=str)
def test_layers_that_compute_the_same_are_patched(kw, interleaved):
    layer = _Layer(pairs=_neighbours if interleaved else _halves, **kw).train()
    weights, state = copy.deepcopy(layer.state_dict()), torch.random.get_rng_state()
    assert patch_attention(torch.nn.ModuleList([layer]), interleaved=interleaved) == 1
    assert layer.training and torch.equal(torch.random.get_rng_state(), state)
    assert all(torch.equal(t, weights[k]) and t.dtype == weights[k].dtype for k, t in layer.state_dict().items())
    assert patch_attention(torch.nn.ModuleList([layer]), interleaved=interleaved) == 1      # and again


def test_rotations_of_part_of_the_channels_are_found_in_the_model_or_its_config():
    model = torch.nn.ModuleList([_Layer(rotary=8)])
    with pytest.raises(ValueError, match="layer 0"):
        patch_attention(_with(_Layer(rotary=8, odd="clip")))
    model.register_buffer("inv_freq", torch.ones(4))
    assert patch_attention(model) == 1
    for attr in ("partial_rotary_factor", "rope_parameters"):
        layer = _Layer(rotary=8)
        setattr(layer.config, attr, 0.5 if attr == "partial_rotary_factor" else {"partial_rotary_factor": 0.5})
        assert patch_attention(_with(layer)) == 2


def _with(layer):
    return torch.nn.ModuleList([_Layer(), layer])


@pytest.mark.parametrize("odd", ["sub_norm", "norm_behind_rotation", "learned_mask", "difference", "cap", "clip", "gate", "sink", "temperature",
                                 "no_rotation", "table_halves"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_layers_whose_own_forward_differs_are_refused_and_none_is_changed(odd, interleaved):
    if odd == "table_halves" and interleaved:
        pytest.skip("taken: test_tables_by_halves_of_interleaved_layers_are_found")
    pairs = _neighbours if interleaved or odd == "table_halves" else _halves
    first, layer = _Layer(pairs=pairs), _Layer(odd, pairs=pairs)
    model = torch.nn.ModuleList([first, layer])
    with pytest.raises(ValueError, match="layer 0"):
        patch_attention(model, interleaved=interleaved)
    assert "forward" not in first.__dict__ and "forward" not in layer.__dict__


@pytest.mark.parametrize("interleaved", [False, True])
def test_the_other_pairing_is_refused(interleaved):
    with pytest.raises(ValueError, match=f"interleaved={not interleaved}"):
        patch_attention(_with(_Layer(pairs=_neighbours if interleaved else _halves)), interleaved=not interleaved)


@pytest.mark.parametrize("config", [dict(sliding_window=8), dict(attn_logit_softcapping=50.0), dict(clip_qkv=8.0), dict(attention_chunk_size=8),
                                    dict(layer_types=["sliding_attention"]), dict(layer_types=["chunked_attention"])], ids=str)
def test_what_only_the_config_says_is_refused(config):
    layer = _Layer()
    layer.config = SimpleNamespace(**config)
    with pytest.raises(ValueError, match="does not know"):
        patch_attention(_with(layer))
    assert "forward" not in layer.__dict__


def test_a_config_with_a_window_that_this_layer_does_not_use():
    one, two, three = _Layer(), _Layer(), _Layer()
    one.config, one.sliding_window = SimpleNamespace(sliding_window=8, layer_types=["full_attention"]), None
    two.config = SimpleNamespace(sliding_window=8, use_sliding_window=False)
    three.config = SimpleNamespace(attention_chunk_size=8, layer_types=["full_attention"])
    assert patch_attention(torch.nn.ModuleList([one, two, three])) == 3


def test_layers_that_cannot_be_compared_are_refused():
    layer = _Layer()
    layer.__class__ = type("Other", (_Layer,), dict(forward=lambda self, tokens: tokens))
    with pytest.raises(ValueError, match="cannot be compared"):
        patch_attention(_with(layer))
    layer = _Layer()
    layer.is_causal = False
    with pytest.raises(ValueError, match="causal"):
        patch_attention(_with(layer))


def test_norms_added_to_a_layer_without_any_are_accepted():
    assert patch_attention(_with(_Layer("norms_unused", head_norms=True))) == 2


def test_tables_by_halves_of_interleaved_layers_are_found(monkeypatch):
    from hira_b200.attention import rope
    seen = []
    monkeypatch.setattr(rope, "hira_attention_forward", lambda *a, **kw: seen.append((kw["interleaved"], kw["table_halves"])))
    model = torch.nn.ModuleList([_Layer(pairs=_neighbours), _Layer("table_halves", pairs=_neighbours, rotary=8)])
    model.register_buffer("inv_freq", torch.ones(4))
    assert patch_attention(model, interleaved=True) == 2
    for m in model:
        m.forward(torch.zeros(1, 1, HIDDEN), (None, None))
    assert seen == [(True, False), (True, True)]
    t = torch.arange(6.0).view(1, 1, 6)
    assert rope._by_channel(t).tolist() == [[[0, 0, 1, 1, 2, 2]]]
