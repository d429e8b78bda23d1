"""Decode attention of several continuations of one prompt.

`hira_decode_attention` searches an index per sequence.  When a batch continues the same prompt many times
(samples of one answer, beams, drafts), the keys its query heads select add up to nearly all of them, and reading
the prompt once for everyone is cheaper than searching it for each: `hira_shared_attention` attends densely to a
prompt kept once and to each sequence's own tail.  `SharedPrompt` keeps the two together;
`HiraCacheLayer.share_prompt` turns a prefilled layer into one.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd import forward_ad

from .. import _lib as L
from .. import index_state as S

_TYPES = (torch.float32, torch.bfloat16)
_plans = {}
_NAMES = ("query", "prefix_keys", "prefix_values", "tail_keys", "tail_values", "prefix_lens", "tail_lens")


def _layout(t: Optional[torch.Tensor]):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.get_device())


def _tail_layout(t: Optional[torch.Tensor]):
    """All but the length, which grows from call to call."""
    if t is None or t.ndim != 4:
        return t if t is None else ()
    b, h, n, d = t.shape
    return b, h, d, min(n, 2), t.stride(), t.dtype, t.get_device()      # the strides of one row need not fit two


def differentiating() -> bool:
    """Whether a derivative of some kind may be asked for at all: one look for calls that need not look at their tensors."""
    return torch.is_grad_enabled() or forward_ad._current_level >= 0


def refuse_grad(what: str, *tensors):
    """The kernels have no backward pass and carry no tangents: a call that would have to be differentiated is refused."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError(f"{what} has no backward pass: call it under torch.no_grad()")
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError(f"{what} has no derivative in forward mode: call it on the primals")


def _lengths(lens, n: int, most: int, device, what: str) -> Optional[torch.Tensor]:
    if lens is None:
        return None
    t = torch.as_tensor(lens)
    if t.shape != (n,) or t.dtype.is_floating_point or t.dtype == torch.bool:
        raise ValueError(f"{what} must be ({n},) whole numbers, got {tuple(t.shape)} {t.dtype}")
    if not t.is_cuda and n and not (0 <= int(t.min()) and int(t.max()) <= most):
        raise ValueError(f"{what} outside 0..{most}: {t.tolist()}")
    if t.is_cuda and t.dtype in (torch.int64, torch.uint32):
        t = t.to(torch.int64).clamp(0, most)          # before 32 bits cut it elsewhere
    return t.to(device=device, dtype=torch.int32).contiguous()


def _check_apart(out, query, named):
    """Rows are read by some blocks while others write theirs: `out` is the query itself, or shares no byte with what is read."""
    for name, t in named:
        if t is not None and torch.is_tensor(t) and t.device == out.device and S.share_memory(out, t) and not (
                t is query and out.data_ptr() == t.data_ptr() and out.shape == t.shape and S.row_strides(out) == S.row_strides(t)):
            raise ValueError(f"out must be memory apart from {name}" + (", or the query itself" if t is query else ""))


def hira_shared_attention(query: torch.Tensor, prefix_keys: torch.Tensor, prefix_values: torch.Tensor,
                          tail_keys: Optional[torch.Tensor] = None, tail_values: Optional[torch.Tensor] = None, *,
                          prefix_lens=None, tail_lens=None, scaling: Optional[float] = None,
                          out: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """query (B, H_q, L_q, D), prefix (P, H_kv, L, D) and (P, H_kv, L, V), tails (B, H_kv, T, D) and (B, H_kv, T, V)
    -> (B, H_q, L_q, V) in the query's type.

    The B = P * n sequences are n continuations of each of P prompts, sequence b of prompt b // n.  Each query
    token attends to its prompt and to its sequence's tail, whose last L_q keys are the query tokens' own: token t
    sees the tail up to T - (L_q - 1 - t).  Without tails there is nothing to hide.

    `prefix_lens` (P,) and `tail_lens` (B,): keys that really are there, in front (what lies behind is not used,
    whatever it holds).  On the host they are checked; on the device they are cut to 0..L and 0..T.  A query that
    sees no key at all gives 0.

    fp32 or bf16, all of one type; D and V multiples of 8 up to 256; B * H_kv up to 65,535.  fp32 is computed in fp32; bf16 with
    fp32 sums and statistics and softmax weights of two bf16 terms (2^-15 of a weight).  Rows have to be contiguous and 16-byte
    aligned: what is not is copied first.  `out` has to be so, and to be the query itself (D = V) or memory apart from all that the call reads.  No backward pass.  A key
    hidden from one query token but not from another has to be finite.

    `status`: a word (int32, on the query's device) that takes the bit HIRA_STATUS_ATTN_FAILED where a kernel gave up on a
    bounded wait; the rows it had are NaN then."""
    if torch.is_grad_enabled() or forward_ad._current_level >= 0:
        refuse_grad("hira_shared_attention", query, prefix_keys, prefix_values, tail_keys, tail_values)
    if scaling is not None:
        scaling = float(scaling)      # a tensor's value, not the tensor, goes with the layout
    if status is not None and (status.dtype != torch.int32 or status.numel() != 1 or status.device != query.device):
        raise ValueError(f"status must be one int32 on {query.device}, got {tuple(status.shape)} {status.dtype} on {status.device}")
    # calls of a layout that has been checked before go straight to the library
    layout = None
    if (tail_keys is None or tail_values is not None and tail_keys.shape[:-1] == tail_values.shape[:-1]) \
            and (prefix_lens is None or torch.is_tensor(prefix_lens) and prefix_lens.is_cuda) \
            and (tail_lens is None or torch.is_tensor(tail_lens) and tail_lens.is_cuda):
        layout = (query.shape, query.stride(), query.dtype, query.get_device(), prefix_keys.shape, prefix_keys.stride(), prefix_keys.dtype,
                  prefix_keys.get_device(), prefix_values.shape, prefix_values.stride(), prefix_values.dtype, prefix_values.get_device(),
                  _tail_layout(tail_keys), _tail_layout(tail_values), _layout(prefix_lens), _layout(tail_lens), _layout(out), scaling)
        plan = _plans.get(layout)
        if plan is not None:
            done = plan(query, prefix_keys, prefix_values, tail_keys, tail_values, prefix_lens, tail_lens, out, status)
            if done is None and out is not None:      # address ranges that meet
                given = (query, prefix_keys, prefix_values, tail_keys, tail_values, prefix_lens, tail_lens)
                _check_apart(out, query, zip(_NAMES, given))
                done = plan(*given, out, status, apart=True)
            if done is not None:
                return done
    if (tail_keys is None) != (tail_values is None):
        raise ValueError("tail_keys and tail_values are given together or not at all")
    named = [("query", query), ("prefix_keys", prefix_keys), ("prefix_values", prefix_values)]
    if tail_keys is not None:
        named += [("tail_keys", tail_keys), ("tail_values", tail_values)]
    elif tail_lens is not None:
        raise ValueError("tail_lens without tails")
    for name, t in named:
        if t.ndim != 4:
            raise ValueError(f"{name} must have 4 dimensions, got {tuple(t.shape)}")
        if t.dtype != query.dtype or t.device != query.device:
            raise ValueError(f"{name} is {t.dtype} on {t.device}, query is {query.dtype} on {query.device}")
    if query.dtype not in _TYPES:
        raise ValueError(f"unsupported dtype {query.dtype}: float32 or bfloat16")
    b, hq, n_q, d = query.shape
    p, h, n, v = prefix_values.shape
    if prefix_keys.shape != (p, h, n, d):
        raise ValueError(f"prefix_keys {tuple(prefix_keys.shape)} fit neither query {tuple(query.shape)} nor prefix_values "
                         f"{tuple(prefix_values.shape)}")
    if p == 0 or b % p:
        raise ValueError(f"{b} sequences are no multiple of {p} prompts")
    if h == 0 or hq % h:
        raise ValueError(f"{hq} query heads are no multiple of {h} key heads")
    if tail_keys is not None and (tail_keys.shape[:2] != (b, h) or tail_keys.shape[3] != d
                                  or tail_values.shape != (b, h, tail_keys.shape[2], v)):
        raise ValueError(f"tails {tuple(tail_keys.shape)} and {tuple(tail_values.shape)} do not fit query {tuple(query.shape)} "
                         f"and prefix_values {tuple(prefix_values.shape)}")
    for name, w in (("D", d), ("V", v)):
        if w % 8 or not 8 <= w <= 256:
            raise ValueError(f"{name}={w} must be a multiple of 8 in 8..256")
    given = (query, prefix_keys, prefix_values, tail_keys, tail_values, prefix_lens, tail_lens)
    prefix_lens = _lengths(prefix_lens, p, n, query.device, "prefix_lens")
    if tail_keys is not None:
        tail_lens = _lengths(tail_lens, b, tail_keys.shape[2], query.device, "tail_lens")
    if out is not None:
        if out.shape != (b, hq, n_q, v) or out.dtype != query.dtype or out.device != query.device or not S.writable_rows(out):
            raise ValueError(f"out must be ({b}, {hq}, {n_q}, {v}) {query.dtype} on {query.device} with aligned contiguous rows")
        _check_apart(out, query, zip(_NAMES, given))
    if not query.is_cuda:
        raise ValueError("hira_shared_attention needs CUDA tensors (there is no CPU fallback)")
    if out is None:
        out = torch.empty((b, hq, n_q, v), dtype=query.dtype, device=query.device)
    if out.numel() == 0:
        return out
    args = tuple(None if t is None else S.with_rows(t) for t in given[:5]) + (prefix_lens, tail_lens)
    plan = S.SharedAttnPlan(*args[:5], d ** -0.5 if scaling is None else scaling, out)
    if layout is not None and all(a is b for a, b in zip(args, given)):
        S.remember(_plans, layout, plan)
    return plan(*args, out, status, apart=True)


def _keep(*tensors):
    """For tensors that may be dropped while the current stream still reads them, another stream's among them."""
    if tensors[0].is_cuda:
        stream = torch.cuda.current_stream(tensors[0].device)
        for t in tensors:
            t.record_stream(stream)


class SharedPrompt:
    """P prompts kept once, and the tails of their P * branches continuations.

        prompt = SharedPrompt(keys, values, branches=16)      # (P, H_kv, L, D), (P, H_kv, L, V)
        prompt.append(k, v)                                   # (P * 16, H_kv, m, D), (P * 16, H_kv, m, V)
        out = prompt.attend(query)                            # (P * 16, H_q, m, D) -> (P * 16, H_q, m, V)
        prompt.reorder(indices)                               # sequence b goes on from what indices[b] was

    Prompts are not copied, unless their rows are not contiguous or not 16-byte aligned.  Tails grow by doubling;
    `max_tail` reserves room for that many tokens, so that nothing moves while a graph that was captured with them
    lives."""

    def __init__(self, prefix_keys: torch.Tensor, prefix_values: torch.Tensor, branches: int, *, prefix_lens=None,
                 max_tail: int = 0, _status: Optional[torch.Tensor] = None):
        for name, t in (("prefix_keys", prefix_keys), ("prefix_values", prefix_values)):
            if t.ndim != 4:
                raise ValueError(f"{name} must have 4 dimensions, got {tuple(t.shape)}")
        if prefix_keys.shape[:3] != prefix_values.shape[:3] or prefix_keys.dtype != prefix_values.dtype \
                or prefix_keys.device != prefix_values.device:
            raise ValueError("prefix_keys and prefix_values must agree in (P, H, L), type and device")
        if branches < 1 or prefix_keys.shape[0] < 1:
            raise ValueError(f"{branches} branches of {prefix_keys.shape[0]} prompts")
        if prefix_keys.dtype not in _TYPES:
            raise ValueError(f"unsupported dtype {prefix_keys.dtype}: float32 or bfloat16")
        self.prefix_keys, self.prefix_values = S.with_rows(prefix_keys), S.with_rows(prefix_values)
        self.prefix_lens = _lengths(prefix_lens, prefix_keys.shape[0], prefix_keys.shape[2], prefix_keys.device, "prefix_lens")
        self.branches = int(branches)
        self.status = torch.zeros((1,), dtype=torch.int32, device=prefix_keys.device) if _status is None else _status
        self._len = 0
        self._k = self._v = None
        self._reserve(max(0, int(max_tail)))

    @property
    def batch(self) -> int:
        return self.prefix_keys.shape[0] * self.branches

    @property
    def tail_len(self) -> int:
        return self._len

    @property
    def tail_keys(self) -> torch.Tensor:
        return self._k[:, :, :self._len]

    @property
    def tail_values(self) -> torch.Tensor:
        return self._v[:, :, :self._len]

    def _reserve(self, rows: int):
        if self._k is not None and rows <= self._k.shape[2]:
            return
        old = None if self._k is None else (self._k, self._v)
        new = []
        for i, like in enumerate((self.prefix_keys, self.prefix_values)):
            t = torch.empty((self.batch, like.shape[1], rows, like.shape[3]), dtype=like.dtype, device=like.device)
            if old is not None:
                t[:, :, :self._len] = old[i][:, :, :self._len]
                _keep(old[i])
            new.append(t)
        self._k, self._v = new
        self._moves = S.RowMoves([(self._k, self._k), (self._v, self._v)])

    def append(self, keys: torch.Tensor, values: torch.Tensor):
        """keys (B, H_kv, m, D), values (B, H_kv, m, V): the next m tokens of every sequence, in the prompts' type and on
        their device."""
        if differentiating():
            refuse_grad("SharedPrompt.append", keys, values)
        for name, t, buf in (("keys", keys, self._k), ("values", values, self._v)):
            if t.ndim != 4 or t.shape[:2] != buf.shape[:2] or t.shape[3] != buf.shape[3] or t.shape[2] != keys.shape[2]:
                raise ValueError(f"{name} {tuple(t.shape)} do not continue tails of {tuple(buf.shape)}")
            if t.dtype != buf.dtype or t.device != buf.device:
                raise ValueError(f"{name} are {t.dtype} on {t.device}, the tails {buf.dtype} on {buf.device}")
        m = keys.shape[2]
        if self._len + m > self._k.shape[2]:
            self._reserve(max(self._len + m, 2 * self._k.shape[2], 16))
        self._k[:, :, self._len:self._len + m] = keys
        self._v[:, :, self._len:self._len + m] = values
        self._len += m
        return self

    def attend(self, query: torch.Tensor, scaling: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """query (B, H_q, m, D), the tokens appended last (or, before the first append, any): see `hira_shared_attention`."""
        k, v = (self.tail_keys, self.tail_values) if self._len else (None, None)
        return hira_shared_attention(query, self.prefix_keys, self.prefix_values, k, v, prefix_lens=self.prefix_lens,
                                     scaling=scaling, out=out, status=self.status)

    def _picks(self, indices) -> torch.Tensor:
        """A sequence continues its own prompt: with several prompts the indices are looked at on the host."""
        idx = S.check_picks(indices, self.batch, self.prefix_keys.device)
        p = self.prefix_keys.shape[0]
        if p > 1:
            host, per = idx.tolist(), idx.numel() // p
            if idx.numel() % p or any(i < 0 or i // self.branches != j // per for j, i in enumerate(host)):
                raise ValueError(f"indices {host} do not keep {p} prompts apart, with equally many sequences each in their order")
        return idx

    def _report(self, idx: torch.Tensor, status: torch.Tensor):
        """What the gather would put into `status`, where there is no tail yet to gather."""
        if idx.is_cuda:
            bad = ((idx < 0) | (idx >= self.batch)).any()
            status.bitwise_or_(bad.to(torch.int32) * L.HIRA_STATUS_BAD_INDEX)

    def reorder(self, indices):
        """In place: sequence b goes on from what sequence indices[b] was (any may be picked many times).  Sequences
        that pick themselves are not touched, and prompts never are.  An index on the device that is out of range
        leaves its sequence as it was and is reported by `check_status`."""
        idx = self._picks(indices)
        if idx.numel() != self.batch:
            raise ValueError(f"{idx.numel()} indices for {self.batch} sequences")
        if self._len:
            S.gather_rows(self._moves, idx, self._len, self.status)
        else:
            self._report(idx, self.status)
        return self

    def select(self, indices) -> "SharedPrompt":
        """The picked sequences (forked where an index repeats, compacted where some are left out) over the same prompts.
        What `check_status` has to report of this one, it has to report of the new one too."""
        idx = self._picks(indices)
        n = idx.numel()
        if n == 0:
            raise ValueError("no sequence picked")
        new = SharedPrompt(self.prefix_keys, self.prefix_values, n // self.prefix_keys.shape[0], max_tail=self._k.shape[2],
                           _status=self.status.clone())
        new.prefix_lens, new._len = self.prefix_lens, self._len
        if self._len:
            S.gather_rows(S.RowMoves([(self._k, new._k), (self._v, new._v)]), idx, self._len, new.status)
        else:
            self._report(idx, new.status)
        _keep(self.status, self._k, self._v)
        return new

    def check_status(self):
        """Raises if an index on the device was out of range, if a kernel of `attend` gave up on a bounded wait, or if the index
        that the prompts come from had something to report (reads one word from the device)."""
        S.raise_for_status(int(self.status.item()))
