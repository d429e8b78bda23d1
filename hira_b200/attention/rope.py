"""Norms of the query and key heads with the position rotation in one pass, and the attention forward that uses it.

`hira_qk_norm_rope` is what a model does between its projections and `HiraCache.update`: an RMS norm of every query
and key head (where the model has one) and the rotation by position, fifteen or so elementwise passes otherwise.
`patch_attention` replaces the forward of a model's attention layers by `hira_attention_forward`: projections,
`hira_qk_norm_rope`, `HiraCache.update`, `hira_attention`, output projection (the hook of examples/patch_llama.py:22-100).
"""
from __future__ import annotations

import copy
from types import MethodType
from typing import Optional

import torch

from .. import index_state as S
from .shared_attention import differentiating, refuse_grad

_TYPES = (torch.float32, torch.bfloat16)
_plans = {}


def _layout(t: torch.Tensor):
    return t.shape, t.stride(), t.dtype, t.get_device()


def _check_apart(query, key, out_q, out_k, reads):
    """Rows are read by many threads while others write: an output is its own input, or shares no byte with what is read or written
    beside it."""
    for name, o, x, other in (("out_q", out_q, query, key), ("out_k", out_k, key, query)):
        if o is None:
            continue
        same = o.data_ptr() == x.data_ptr() and S.row_strides(o) == S.row_strides(x)
        if not same and S.share_memory(o, x) or S.share_memory(o, other):
            raise ValueError(f"{name} must be its own input or memory apart from both inputs")
        for what, t in reads:
            if t is not None and S.share_memory(o, t):
                raise ValueError(f"{name} must be memory apart from {what}")
    if out_q is not None and out_k is not None and S.share_memory(out_q, out_k):
        raise ValueError("out_q and out_k are the same memory, at least in part")


def _table(t: torch.Tensor, b: int, n: int, name: str) -> torch.Tensor:
    if t.ndim == 2:
        t = t.unsqueeze(0)
    if t.ndim != 3 or t.shape[0] not in (1, b) or t.shape[1] != n:
        raise ValueError(f"{name} must be ({b} or 1, {n}, R) or ({n}, R), got {tuple(t.shape)}")
    if t.dtype not in _TYPES:
        t = t.float()
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def hira_qk_norm_rope(query: torch.Tensor, key: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, *,
                      q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                      interleaved: bool = False, out_q: Optional[torch.Tensor] = None, out_k: Optional[torch.Tensor] = None):
    """query (B, H_q, L, D), key (B, H_kv, L, D) -> the two normalised and rotated, in their type.

    `cos`, `sin` (B or 1, L, R) or (L, R), R <= D even: tables with the factors of each of the first R channels at that
    channel's own place; channels i and i + R/2 form a pair, or 2i and 2i + 1 when `interleaved`.  (Some models that pair
    2i and 2i + 1 hand out tables with the pair's value at i and i + R/2: those have to be laid out by channel first, as
    `hira_attention_forward` does with `table_halves`.)  The channels behind R are not rotated.  `q_weight` / `k_weight`
    (D,): RMS norm of that side's heads with this weight; None: no norm.  Computed in fp32 and rounded once.

    fp32 or bf16; D a multiple of 8 up to 256.  Any strides with contiguous, 16-byte aligned rows (a projection's
    transposed view as it is); others are copied.  `out_q` / `out_k`: where to write, with such rows: the input itself,
    or memory apart from all that the call reads and from one another (part of a cache, say; the heads of one projection
    are apart although they lie between each other).  No backward pass."""
    if differentiating():
        refuse_grad("hira_qk_norm_rope", query, key, q_weight, k_weight, cos, sin)
    eps, interleaved = float(eps), bool(interleaved)
    # calls of a layout that has been checked before go straight to the library
    layout = (query.shape, query.stride(), query.dtype, query.get_device(), key.shape, key.stride(), key.dtype, key.get_device(),
              cos.shape, cos.stride(), cos.dtype, cos.get_device(), sin.shape, sin.stride(), sin.dtype, sin.get_device(),
              None if q_weight is None else _layout(q_weight), None if k_weight is None else _layout(k_weight),
              None if out_q is None else _layout(out_q), None if out_k is None else _layout(out_k), eps, interleaved)
    plan = _plans.get(layout)
    if plan is not None:
        done = plan(query, key, cos, sin, q_weight, k_weight, out_q, out_k)
        if done is None and (out_q is not None or out_k is not None):      # address ranges that meet
            _check_apart(query, key, out_q, out_k, (("cos", cos), ("sin", sin), ("q_weight", q_weight), ("k_weight", k_weight)))
            done = plan(query, key, cos, sin, q_weight, k_weight, out_q, out_k, apart=True)
        if done is not None:
            return done
    if query.ndim != 4 or key.ndim != 4:
        raise ValueError(f"query and key must be (B, H, L, D), got {tuple(query.shape)} and {tuple(key.shape)}")
    b, hq, n, d = query.shape
    if key.shape[0] != b or key.shape[2] != n or key.shape[3] != d:
        raise ValueError(f"key {tuple(key.shape)} does not go with query {tuple(query.shape)}")
    if query.dtype not in _TYPES or key.dtype != query.dtype:
        raise ValueError(f"query is {query.dtype}, key {key.dtype}: both float32 or both bfloat16")
    if d % 8 or not 8 <= d <= 256:
        raise ValueError(f"D={d} must be a multiple of 8 in 8..256")
    for name, t in (("key", key), ("cos", cos), ("sin", sin), ("q_weight", q_weight), ("k_weight", k_weight), ("out_q", out_q),
                    ("out_k", out_k)):
        if t is not None and t.device != query.device:
            raise ValueError(f"{name} is on {t.device}, query on {query.device}")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and (w.shape != (d,) or w.dtype != query.dtype):
            raise ValueError(f"{name} must be ({d},) {query.dtype}, got {tuple(w.shape)} {w.dtype}")
    given = cos, sin
    cos, sin = _table(cos, b, n, "cos"), _table(sin, b, n, "sin")
    if cos.shape[2] != sin.shape[2] or cos.dtype != sin.dtype:
        raise ValueError(f"cos {tuple(cos.shape)} {cos.dtype} and sin {tuple(sin.shape)} {sin.dtype} differ")
    r = cos.shape[2]
    if r % 2 or r > d:
        raise ValueError(f"{r} rotated channels: must be even and at most {d}")
    for name, o, x in (("out_q", out_q, query), ("out_k", out_k, key)):
        if o is None:
            continue
        if o.shape != x.shape or o.dtype != x.dtype or not S.writable_rows(o):
            raise ValueError(f"{name} must be {tuple(x.shape)} {x.dtype} with aligned contiguous rows")
    _check_apart(query, key, out_q, out_k, (("cos", given[0]), ("sin", given[1]), ("q_weight", q_weight), ("k_weight", k_weight)))
    if not query.is_cuda:
        raise ValueError("hira_qk_norm_rope needs CUDA tensors (there is no CPU fallback)")
    args = (S.with_rows(query), S.with_rows(key), cos, sin, *(None if w is None else S.aligned(w.contiguous()) for w in (q_weight, k_weight)))
    as_given = all(a is b for a, b in zip(args, (query, key, *given, q_weight, k_weight)))
    oq = torch.empty((b, hq, n, d), dtype=query.dtype, device=query.device) if out_q is None else out_q
    ok = torch.empty(tuple(key.shape), dtype=key.dtype, device=key.device) if out_k is None else out_k
    plan = S.RopePlan(*args[:4], eps, interleaved, oq, ok)
    if as_given:
        S.remember(_plans, layout, plan)
    return plan(*args, oq, ok, apart=True)


def _by_channel(t: torch.Tensor) -> torch.Tensor:
    """A table that holds pair i's value at i (and again at i + R/2) as one that holds it at 2i and 2i + 1."""
    return t[..., :t.shape[-1] // 2].unsqueeze(-1).expand(*t.shape[:-1], t.shape[-1] // 2, 2).flatten(-2)


def hira_attention_forward(module, hidden_states: torch.Tensor, position_embeddings, attention_mask: Optional[torch.Tensor] = None,
                           past_key_values=None, hira_config=None, interleaved: bool = False, table_halves: bool = False, **kwargs):
    """Forward of a decoder's attention layer over a HiraCache.  `module` has q_proj, k_proj, v_proj, o_proj, head_dim
    and layer_idx, and may have q_norm and k_norm (RMS norms of single heads: `weight` (head_dim,) and an epsilon).
    `table_halves`: the model pairs channels 2i and 2i + 1 (`interleaved`), but its tables hold the pair's value at i and
    i + R/2, as if it paired those."""
    from .hira_attention import hira_attention
    if past_key_values is None:
        raise ValueError("hira_attention_forward needs a HiraCache as past_key_values")
    b, n, _ = hidden_states.shape

    def heads(proj):
        return proj(hidden_states).view(b, n, -1, module.head_dim).transpose(1, 2)
    q, k, v = heads(module.q_proj), heads(module.k_proj), heads(module.v_proj)
    q_norm, k_norm = getattr(module, "q_norm", None), getattr(module, "k_norm", None)
    cos, sin = position_embeddings
    if interleaved and table_halves:
        cos, sin = _by_channel(cos), _by_channel(sin)
    eps = {getattr(m, "variance_epsilon", getattr(m, "eps", None)) for m in (q_norm, k_norm) if m is not None}
    if len(eps) > 1:
        raise ValueError(f"q_norm and k_norm have different epsilons: {sorted(eps)}")
    q, k = hira_qk_norm_rope(q, k, cos, sin, q_weight=None if q_norm is None else q_norm.weight,
                             k_weight=None if k_norm is None else k_norm.weight, eps=eps.pop() if eps else 1e-6,
                             interleaved=interleaved)
    cache_output, _ = past_key_values.update(k, v, module.layer_idx)
    out, _ = hira_attention(module, q, cache_output, None, attention_mask, scaling=getattr(module, "scaling", None),
                            hira_config=hira_config)
    return module.o_proj(out.reshape(b, n, -1)), None


def _is_head_rms_norm(norm, width: int) -> bool:
    """Whether `norm` computes x * rsqrt(mean(x^2) + eps) * weight over `width` channels, seen from what it makes of a vector
    (a norm about the mean, or with weights about one, does not)."""
    w, eps = getattr(norm, "weight", None), getattr(norm, "variance_epsilon", getattr(norm, "eps", None))
    if w is None or eps is None or tuple(w.shape) != (width,):
        return False
    x = torch.linspace(-1.0, 2.0, width, device=w.device, dtype=torch.float32)
    with torch.no_grad():
        got = norm(x.to(w.dtype)).double()
    want = x.double() * torch.rsqrt(x.double().square().mean() + eps) * w.double()
    # three roundings of x, x^ and the product, in the weight's type
    return bool(((got - want).abs() <= 2 * torch.finfo(w.dtype).eps * want.abs() + 1e-6).all())


_PARTS = ("q_proj", "k_proj", "v_proj", "o_proj", "q_norm", "k_norm")


def _known_difference(m) -> Optional[str]:
    """What a layer says of itself that a HiraCache's attention does not do: where it stands on the layer, and where the layer
    has no word of its own, in its config (whose mask or kernel arguments a single forward does not show)."""
    config = getattr(m, "config", None)
    for name in ("sliding_window", "attention_chunk_size", "attn_logit_softcapping", "sinks", "clip_qkv"):
        if name == "sliding_window" and not hasattr(m, name) and not getattr(config, "use_sliding_window", True):
            continue
        if (getattr(m, name) if hasattr(m, name) else getattr(config, name, None) if name != "attention_chunk_size" else None) is not None:
            return f"has {name}, which a HiraCache's attention does not know"
    types = getattr(config, "layer_types", None)
    if types is not None and isinstance(m.layer_idx, int) and m.layer_idx < len(types) \
            and types[m.layer_idx] not in ("full_attention", "attention", "hybrid"):
        return f"is of type {types[m.layer_idx]}, which a HiraCache's attention does not know"
    if types is None and getattr(config, "attention_chunk_size", None) is not None:
        return "has attention_chunk_size, which a HiraCache's attention does not know"
    if not getattr(m, "use_rope", True):
        return "does not rotate its heads"
    if not getattr(m, "is_causal", True):
        return "is not causal"
    for name, _ in (*m.named_parameters(), *m.named_buffers()):
        if name.split(".")[0] not in _PARTS and "inv_freq" not in name:      # frequencies: the rotation is compared anyway
            return f"has {name}, which hira_attention_forward does not use"
    return None


def _rotated(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, interleaved: bool) -> torch.Tensor:
    """The rotation of `hira_qk_norm_rope`, in elementary operations."""
    r = cos.shape[-1]
    t = x[..., :r]
    if interleaved:
        other = torch.stack([-t[..., 1::2], t[..., 0::2]], dim=-1).flatten(-2)
    else:
        other = torch.cat([-t[..., r // 2:], t[..., :r // 2]], dim=-1)
    return torch.cat([t * cos[:, None] + other * sin[:, None], x[..., r:]], dim=-1)


def _plain_forward(m, x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, interleaved: bool, norms: bool) -> torch.Tensor:
    """What `hira_attention_forward` makes of a prompt, in elementary operations; cos None: the scores before rotation and softmax."""
    b, n, _ = x.shape
    q, k, v = (proj(x).view(b, n, -1, m.head_dim).transpose(1, 2) for proj in (m.q_proj, m.k_proj, m.v_proj))
    if norms:
        q, k = (t if norm is None else norm(t) for t, norm in ((q, getattr(m, "q_norm", None)), (k, getattr(m, "k_norm", None))))
    if cos is not None:
        q, k = _rotated(q, cos, sin, interleaved), _rotated(k, cos, sin, interleaved)
    scaling = getattr(m, "scaling", None)
    s = (m.head_dim ** -0.5 if scaling is None else scaling) * (q @ k.repeat_interleave(q.shape[1] // k.shape[1], dim=1).transpose(-1, -2))
    if cos is None:
        return s
    s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=x.device).triu(1), float("-inf"))
    o = torch.softmax(s, dim=-1) @ v.repeat_interleave(q.shape[1] // v.shape[1], dim=1)
    return m.o_proj(o.transpose(1, 2).reshape(b, n, -1))


@torch.no_grad()
def _own_forward_differs(layer, widths, interleaved: bool, table_halves: bool) -> Optional[str]:
    """Runs a copy of the layer with the forward of its class and with `_plain_forward` on a few random tokens in 64 bits, and
    says what is wrong where they disagree.  The tables have a value of its own for every channel, so that another pairing of
    the channels, or another use of the tables, shows; logits of about 2 and of about 200, so that a cap or a clip shows.
    `widths`: numbers of rotated channels that the model may use.  A layer without a forward has nothing to disagree with."""
    own = type(layer).forward
    if own is torch.nn.Module.forward:
        return None
    why = None
    try:
        m = copy.deepcopy(layer).double().eval()
        if hasattr(getattr(m, "config", None), "_attn_implementation"):
            m.config._attn_implementation = "eager"
        w, n = m.q_proj.weight, 7
        g = torch.Generator().manual_seed(1)

        def rnd(*shape):
            return torch.randn(shape, generator=g, dtype=torch.float64).to(w.device)
        x = rnd(1, n, w.shape[1])
        mask = torch.full((1, 1, n, n), torch.finfo(torch.float64).min, dtype=torch.float64, device=w.device).triu(1)
        std = float(_plain_forward(m, x, None, None, interleaved, True).std())
        for r in widths:
            cos, sin = rnd(1, n, r).tanh(), rnd(1, n, r).tanh()
            # norms that were added to a layer whose own forward has none are `hira_attention_forward`'s to apply
            equal = {True: True, False: getattr(m, "q_norm", None) is not None or getattr(m, "k_norm", None) is not None}
            try:
                for logit in (2.0, 200.0):
                    y = x * (min(max((logit / std) ** 0.5, 1e-3), 1e3) if std > 0 else 1.0)
                    got = own(m, hidden_states=y, position_embeddings=(cos, sin), attention_mask=mask, past_key_values=None)
                    got = got[0] if isinstance(got, (tuple, list)) else got
                    tables = (_by_channel(cos), _by_channel(sin)) if table_halves else (cos, sin)
                    for norms in equal:
                        want = _plain_forward(m, y, *tables, interleaved, norms)
                        # layers do parts of this in 32 bits: 2^-24 of logits of some 1000, more than ten times over
                        equal[norms] = equal[norms] and bool(((got - want).norm() <= 1e-3 * want.norm() + 1e-30))
            except Exception as e:          # of this width; whatever a class's forward may raise
                why = why or f"cannot be compared with its own forward ({type(e).__name__}: {e})"
                continue
            if any(equal.values()):
                return None
            why = "computes something else than hira_attention_forward"
    except Exception as e:
        why = f"cannot be compared with its own forward ({type(e).__name__}: {e})"
    return why


def _rotary_widths(model, m) -> list:
    """How many channels a layer may rotate: as its model's tables say, as its config says, all."""
    widths = [2 * b.numel() for name, b in model.named_buffers() if name.split(".")[-1] == "inv_freq"]
    config = getattr(m, "config", None)
    for src in (getattr(config, "rope_parameters", None) or {}, getattr(config, "__dict__", {})):
        if src.get("partial_rotary_factor"):
            widths.append(int(m.head_dim * src["partial_rotary_factor"]))
    return [r for r in dict.fromkeys([*widths, m.head_dim]) if 0 < r <= m.head_dim and r % 2 == 0]


def patch_attention(model, hira_config=None, *, interleaved: bool = False) -> int:
    """Gives every attention layer of `model` (a module with q_proj, k_proj, v_proj, o_proj, head_dim and layer_idx)
    `hira_attention_forward` as its forward; returns how many there were.  Run the model under `torch.no_grad()` with
    a HiraCache as `past_key_values`.  `interleaved`: how the model pairs the channels it rotates.  How the tables of an
    interleaved model are laid out (`hira_attention_forward`'s `table_halves`) is found out from its layers.

    A layer that computes something else is refused, and then no layer is changed: sliding windows, chunks, capped logits, sinks,
    no rotation, other norms than RMS norms of single heads, parameters that the new forward does not use; and any layer whose
    own forward disagrees with the new one on a few random tokens, which are run in 64 bits on a copy of each layer (another
    pairing of the channels than `interleaved` says is found that way).  q_norm and k_norm that were added to a layer whose own
    forward has none are applied."""
    layers = [m for m in model.modules()
              if all(hasattr(m, a) for a in ("q_proj", "k_proj", "v_proj", "o_proj", "head_dim", "layer_idx"))]
    if not layers:
        raise ValueError("the model has no attention layer with q_proj, k_proj, v_proj, o_proj, head_dim and layer_idx")
    halves = []
    for m in layers:
        why = _known_difference(m)
        if why is None:
            for name in ("q_norm", "k_norm"):
                norm = getattr(m, name, None)
                if norm is not None and not _is_head_rms_norm(norm, m.head_dim):
                    raise ValueError(f"{name} of layer {m.layer_idx} is no RMS norm of single heads")
            widths = _rotary_widths(model, m)
            why = _own_forward_differs(m, widths, bool(interleaved), False)
            halves.append(bool(interleaved and why and _own_forward_differs(m, widths, True, True) is None))
            if halves[-1]:
                why = None
        if why is not None:
            raise ValueError(f"layer {m.layer_idx} {why}" + (f" with interleaved={bool(interleaved)}" if "something else" in why else ""))
    for m, by_half in zip(layers, halves):
        def forward(self, hidden_states, position_embeddings=None, attention_mask=None, past_key_values=None, _halves=by_half, **kwargs):
            return hira_attention_forward(self, hidden_states, position_embeddings, attention_mask, past_key_values,
                                          hira_config=hira_config, interleaved=interleaved, table_halves=_halves, **kwargs)
        m.forward = MethodType(forward, m)
    return len(layers)
