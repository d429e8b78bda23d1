"""What the operators for several continuations refuse, and what the host decides, on the CPU."""
import ctypes as C

import pytest
import torch

from hira_b200 import CUDAIndexer, SharedPrompt, hira_qk_norm_rope, hira_shared_attention, patch_attention
from hira_b200 import _lib as L
from hira_b200 import index_state as S


def _t(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype)


GOOD = dict(query=(6, 4, 1, 64), prefix_keys=(2, 2, 9, 64), prefix_values=(2, 2, 9, 64), tail_keys=(6, 2, 3, 64), tail_values=(6, 2, 3, 64))


@pytest.mark.parametrize("change,match", [
    (dict(query=(6, 4, 64)), "4 dimensions"), (dict(prefix_keys=(2, 2, 8, 64)), "fit neither"), (dict(prefix_keys=(2, 2, 9, 72)), "fit neither"),
    (dict(query=(5, 4, 1, 64), tail_keys=(5, 2, 3, 64), tail_values=(5, 2, 3, 64)), "no multiple"), (dict(query=(6, 3, 1, 64)), "no multiple"),
    (dict(tail_keys=(6, 2, 4, 64)), "do not fit"), (dict(tail_values=(6, 2, 3, 72)), "do not fit"), (dict(tail_keys=(3, 2, 3, 64)), "do not fit"),
    (dict(query=(6, 4, 1, 60), prefix_keys=(2, 2, 9, 60), tail_keys=(6, 2, 3, 60)), "multiple of 8"),
    (dict(prefix_values=(2, 2, 9, 264), tail_values=(6, 2, 3, 264)), "multiple of 8"), (dict(tail_keys=None), "together"), ({}, "CUDA"),
])
def test_shared_attention_refuses(change, match):
    shapes = {**GOOD, **change}
    with pytest.raises(ValueError, match=match):
        hira_shared_attention(**{k: None if s is None else _t(*s) for k, s in shapes.items()})


def test_shared_attention_refuses_types_lengths_and_gradients():
    a = {k: _t(*s) for k, s in GOOD.items()}
    with pytest.raises(ValueError, match="query is"):
        hira_shared_attention(**{**a, "tail_keys": a["tail_keys"].float()})
    with pytest.raises(ValueError, match="unsupported dtype"):
        hira_shared_attention(**{k: t.half() for k, t in a.items()})
    for kw, match in ((dict(prefix_lens=[9, 10]), "outside"), (dict(prefix_lens=[-1, 1]), "outside"), (dict(prefix_lens=[1]), "whole numbers"),
                      (dict(tail_lens=[1.0] * 6), "whole numbers"), (dict(tail_lens=[4] * 6), "outside")):
        with pytest.raises(ValueError, match=match):
            hira_shared_attention(**a, **kw)
    with pytest.raises(ValueError, match="without tails"):
        hira_shared_attention(a["query"], a["prefix_keys"], a["prefix_values"], tail_lens=[0] * 6)
    with pytest.raises(ValueError, match="no backward"):
        hira_shared_attention(**{**a, "query": a["query"].float().requires_grad_().bfloat16()})


@pytest.mark.parametrize("kw,match", [
    (dict(key=(2, 2, 5, 64)), "does not go"), (dict(key=(2, 2, 4, 72)), "does not go"), (dict(cos=(3, 4, 64)), "must be"), (dict(cos=(2, 5, 64)), "must be"),
    (dict(cos=(2, 4, 32)), "differ"), (dict(cos=(2, 4, 7), sin=(2, 4, 7)), "even"), (dict(cos=(2, 4, 66), sin=(2, 4, 66)), "at most"),
    (dict(q_weight=(32,)), "q_weight"), (dict(query=(2, 4, 4, 60), key=(2, 2, 4, 60)), "multiple of 8"), ({}, "CUDA"),
])
def test_rotation_refuses(kw, match):
    shapes = {**dict(query=(2, 4, 4, 64), key=(2, 2, 4, 64), cos=(2, 4, 64), sin=(2, 4, 64)), **kw}
    with pytest.raises(ValueError, match=match):
        hira_qk_norm_rope(**{k: _t(*s) for k, s in shapes.items()})


def test_rotation_refuses_types_and_outputs():
    q, k, c = _t(2, 4, 4, 64), _t(2, 2, 4, 64), _t(2, 4, 64)
    for kw, match in ((dict(q_weight=torch.ones(64)), "q_weight"), (dict(out_q=q.float()), "out_q"), (dict(out_k=k[:, :1].expand(2, 2, 4, 64)), "out_k"),
                      (dict(out_q=q.transpose(1, 2).contiguous().transpose(1, 2)[..., :32]), "out_q"), (dict(out_q=q.flip(0).view(2, 4, 4, 64)), "CUDA")):
        with pytest.raises(ValueError, match=match):
            hira_qk_norm_rope(q, k, c, c, **kw)
    buf = _t(2, 6, 5, 64)
    with pytest.raises(ValueError, match="apart"):       # one row off: rows would be overwritten before they are read
        hira_qk_norm_rope(buf[:, :4, :4], buf[:, 4:, :4], c, c, out_q=buf[:, :4, 1:])
    same = _t(2, 4, 4, 64)
    with pytest.raises(ValueError, match="same memory"):
        hira_qk_norm_rope(q, k, c, c, out_q=same, out_k=same[:, :2])
    with pytest.raises(ValueError, match="query is"):
        hira_qk_norm_rope(q, k.float(), c, c)
    with pytest.raises(ValueError, match="no backward"):
        hira_qk_norm_rope(q.float().requires_grad_(), k.float(), c, c)
    with pytest.raises(ValueError, match="no attention layer"):
        patch_attention(torch.nn.Linear(2, 2))


@pytest.mark.parametrize("picks,match", [([0, 3], "outside"), ([-1], "outside"), ([[0]], "one-dimensional"), ([0.5], "whole"), ([True, False], "mask")])
def test_picks_are_checked_on_the_host(picks, match):
    with pytest.raises(ValueError, match=match):
        S.check_picks(picks, 3, "cpu")
    assert S.check_picks([True, False, True], 3, "cpu").tolist() == [0, 2]
    assert S.check_picks(torch.tensor([2, 0], dtype=torch.int32), 3, "cpu").dtype == torch.int64


def test_shared_prompt_refuses():
    k = _t(2, 2, 9, 64)
    for args, match in (((k, k, 0), "branches"), ((k, _t(2, 2, 8, 64), 2), "agree"), ((k, k.float(), 2), "agree"), ((k.half(), k.half(), 2), "unsupported"),
                        ((k[0], k, 2), "4 dimensions")):
        with pytest.raises(ValueError, match=match):
            SharedPrompt(*args)
    p = SharedPrompt(k, k, 3, max_tail=2)
    for shape in ((6, 2, 1, 72), (5, 2, 1, 64), (6, 1, 1, 64)):
        with pytest.raises(ValueError, match="do not continue"):
            p.append(_t(*shape), _t(*shape))
    with pytest.raises(ValueError, match="do not continue"):
        p.append(_t(6, 2, 1, 64), _t(6, 2, 2, 64))
    for n in (1, 1, 5, 20):
        p.append(torch.full((6, 2, n, 64), float(n)).bfloat16(), _t(6, 2, n, 64))
    assert p.tail_len == 27 and p.tail_keys[0, 0, :, 0].tolist() == [1.0] * 2 + [5.0] * 5 + [20.0] * 20
    for picks, match in (([0, 1, 2, 3, 4], "apart"), ([0, 1, 2], "apart"), ([3, 4, 5, 0, 1, 2], "apart"), ([], "picked")):
        with pytest.raises(ValueError, match=match):
            p.select(picks)
    with pytest.raises(ValueError, match="indices for"):
        p.reorder([0, 3])


def test_an_index_that_is_not_built_cannot_be_picked_from():
    for f in (CUDAIndexer(3, 1, 8).reorder, CUDAIndexer(3, 1, 8).select):
        with pytest.raises(ValueError, match="not built"):
            f([0])


def _args(**kw):
    a = L.HiraSharedAttnStruct()
    for n in ("q", "prefix_k", "prefix_v", "tail_k", "tail_v", "out"):
        setattr(a, n, 1 << 20)
    for n, v in dict(dtype=L.HIRA_BF16, n_prompts=1, n_branches=2, n_kv=2, group=2, n_q=1, dim=64, vdim=64, prefix_len=10, tail_len=3).items():
        setattr(a, n, v)
    for n, v in kw.items():
        if isinstance(v, tuple):
            getattr(a, n)[:] = v
        else:
            setattr(a, n, v)
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=7), L.HIRA_ERR_DTYPE), (dict(n_kv=0), L.HIRA_ERR_SHAPE), (dict(dim=60), L.HIRA_ERR_SHAPE), (dict(vdim=264), L.HIRA_ERR_SHAPE),
    (dict(prefix_len=-1), L.HIRA_ERR_SHAPE), (dict(n_branches=1 << 20), L.HIRA_ERR_SHAPE), (dict(q=None), L.HIRA_ERR_ARG),
    (dict(prefix_v=None), L.HIRA_ERR_ARG), (dict(tail_k=None), L.HIRA_ERR_ARG), (dict(q=(1 << 20) + 8), L.HIRA_ERR_ARG),
    (dict(tail_v_stride=(0, 4, 64)), L.HIRA_ERR_ARG), ({}, L.HIRA_ERR_CAPACITY),
])
def test_library_refuses_before_any_launch(kw, code):
    lib, a = L.load(), _args(**kw)
    need = lib.hira_shared_attn_workspace_bytes(C.byref(a))
    assert (need > 0) == (code == L.HIRA_ERR_CAPACITY)
    assert lib.hira_shared_attn(C.byref(a), None, 0, None) == code and lib.hira_last_error()
    assert lib.hira_shared_attn(None, None, 0, None) == L.HIRA_ERR_ARG


def test_library_refuses_gathers_that_do_not_fit():
    lib, item = L.load(), L.HiraGatherItemStruct
    one = lambda **kw: (item * 1)(item(**{**dict(src=4096, dst=8192, n_seg=1, bytes=16, bytes_filled=16), **kw}))
    for items, n, src, dst, place, code in (
            (one(), 1, 2, 3, 1, L.HIRA_ERR_SHAPE), (one(), 1, 0, 1, 0, L.HIRA_ERR_SHAPE), (one(), 1, 2049, 1, 0, L.HIRA_ERR_SHAPE),
            (one(), 25, 1, 1, 0, L.HIRA_ERR_SHAPE), (one(bytes=32), 1, 1, 1, 0, L.HIRA_ERR_SHAPE), (one(), 1, 1, 1, 1, L.HIRA_ERR_ARG),
            (one(dst=4096), 1, 1, 1, 0, L.HIRA_ERR_ARG), (one(bytes=14), 1, 1, 1, 0, L.HIRA_ERR_ARG), (one(src=None), 1, 1, 1, 0, L.HIRA_ERR_ARG)):
        assert lib.hira_gather(items, n, 4096, src, dst, place, None, None) == code and lib.hira_last_error()
    assert lib.hira_gather(None, 1, 4096, 1, 1, 0, None, None) == L.HIRA_ERR_ARG
    assert lib.hira_gather(one(n_seg=0), 1, 4096, 1, 1, 0, None, None) == L.HIRA_OK      # nothing to move
    a = S.IndexState(n_heads=4, dim=64, vdim=64, bf=8, depth=2, cap_parents=16, dtype=torch.float32, vdtype=torch.float32, device="cpu")
    b = S.IndexState(n_heads=6, dim=64, vdim=64, bf=8, depth=2, cap_parents=17, dtype=torch.float32, vdtype=torch.float32, device="cpu")
    assert lib.hira_gather_index(a.struct, b.struct, 2, 3, 4096, None, 0, None, None, None) == L.HIRA_ERR_SHAPE
    assert lib.hira_gather_index(a.struct, a.struct, 3, 3, 4096, None, 0, None, None, None) == L.HIRA_ERR_SHAPE


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=5), L.HIRA_ERR_DTYPE), (dict(table_dtype=5), L.HIRA_ERR_DTYPE), (dict(dim=12), L.HIRA_ERR_SHAPE), (dict(rotary=65), L.HIRA_ERR_SHAPE),
    (dict(rotary=72), L.HIRA_ERR_SHAPE), (dict(batch=65536), L.HIRA_ERR_SHAPE), (dict(k=None), L.HIRA_ERR_ARG), (dict(sin=None), L.HIRA_ERR_ARG),
    (dict(q_out=4100), L.HIRA_ERR_ARG), (dict(batch=0), L.HIRA_OK), (dict(n_tokens=0), L.HIRA_OK),
])
def test_library_refuses_rotations_that_do_not_fit(kw, code):
    a = L.HiraRopeStruct(q=4096, k=8192, q_out=4096, k_out=8192, cos=512, sin=1024, dtype=0, table_dtype=0, batch=1, n_tokens=1, q_heads=1,
                         k_heads=1, dim=64, rotary=64, eps=1e-6)
    for n, v in kw.items():
        setattr(a, n, v)
    assert L.load().hira_qk_norm_rope(C.byref(a), None) == code


def test_rotation_refuses_to_overwrite_heads_that_are_queries_and_keys_at_once():
    x, c = _t(2, 4, 4, 64), _t(2, 4, 64)
    for kw in (dict(out_q=x), dict(out_k=x)):
        with pytest.raises(ValueError, match="apart"):
            hira_qk_norm_rope(x, x, c, c, **kw)


def test_shared_prompt_copies_rows_that_are_not_aligned_once():
    k = torch.randn(2, 2, 9, 64).bfloat16()
    flat = torch.cat([k.new_zeros(1), k.flatten()])
    odd = flat[1:].view(k.shape)
    p = SharedPrompt(odd, k, 2)
    assert p.prefix_values is k and p.prefix_keys is not odd and torch.equal(p.prefix_keys, k)
    assert S.row_strides(p.prefix_keys) is not None


@pytest.mark.parametrize("name,value", [("sliding_window", 4096), ("attn_logit_softcapping", 50.0), ("sinks", torch.zeros(4)), ("use_rope", False)])
def test_layers_that_compute_something_else_are_not_patched(name, value):
    layer = torch.nn.Module()
    for proj in ("q_proj", "k_proj", "v_proj", "o_proj"):
        setattr(layer, proj, torch.nn.Linear(8, 8))
    layer.head_dim, layer.layer_idx, layer.sliding_window = 8, 0, None
    model, before = torch.nn.ModuleList([layer]), layer.forward
    setattr(layer, name, value)
    with pytest.raises(ValueError, match="layer 0"):
        patch_attention(model)
    assert layer.forward == before
    setattr(layer, name, None if name != "use_rope" else True)
    assert patch_attention(model) == 1


@pytest.mark.parametrize("on", [True, False])
def test_a_forked_state_uses_the_int8_copy_only_if_its_source_does(on):
    a = S.IndexState(n_heads=2, dim=128, vdim=128, bf=8, depth=2, cap_parents=16, dtype=torch.float32, vdtype=torch.float32, device="cpu",
                     int8_copy=True)
    a.enable_int8_copy(on)
    b = a.like(6)
    assert all(bool(getattr(b._struct, n)) == on for n in S.IndexState.Q8_ARRAYS) and b.children_q8.shape[0] == 6
    b.enable_int8_copy(True)
    assert b._struct.children_q8 == b.children_q8.data_ptr() and bool(a._struct.children_q8) == on


@pytest.mark.parametrize("on", [True, False])
def test_a_grown_state_uses_the_int8_copy_only_if_it_did_before(on):
    a = S.IndexState(n_heads=2, dim=128, vdim=128, bf=8, depth=2, cap_parents=16, dtype=torch.float32, vdtype=torch.float32, device="cpu",
                     int8_copy=True)
    a.enable_int8_copy(on)
    b = a.grown(32)
    assert b.cap_parents == 32 and all(bool(getattr(b._struct, n)) == on for n in S.IndexState.Q8_ARRAYS)


def test_rotation_refuses_outputs_that_overlap_what_is_read_or_written_beside_them():
    c = _t(2, 4, 64)
    q, k, buf = _t(2, 4, 4, 64), _t(2, 2, 4, 64), _t(2, 8, 4, 64)
    for kw, match in ((dict(out_q=buf[:, :4], out_k=buf[:, 3:5]), "same memory"),
                      (dict(query=buf[:, :4], key=buf[:, 1:3], out_q=buf[:, :4]), "apart"),
                      (dict(query=buf[:, :4], key=buf[:, 3:5], out_k=buf[:, 3:5]), "apart"),
                      (dict(out_q=buf[:, :4], cos=buf[:, 2, :, :]), "apart from cos"),
                      (dict(out_k=buf[:, :2], k_weight=buf[0, 1, 3]), "apart from k_weight"),
                      (dict(query=buf[:, :4], key=buf[:, 4:6], out_q=buf[:, 4:]), "apart"),
                      (dict(out_q=buf.flatten().as_strided((2, 4, 4, 64), (2048, 64, 64, 1))), "out_q must be")):
        with pytest.raises(ValueError, match=match):
            hira_qk_norm_rope(**{**dict(query=q, key=k, cos=c, sin=c), **kw})
    # heads of one projection lie between each other, and part of a buffer beside them: all of them apart
    fused, tokens = _t(2, 4, 10, 64).transpose(1, 2), _t(2, 9, 6, 64)
    for kw in (dict(query=fused[:, :4], key=fused[:, 4:6], out_q=fused[:, :4], out_k=fused[:, 4:6]),
               dict(query=fused[:, :4], key=fused[:, 4:6], out_q=fused[:, 6:], out_k=fused[:, 4:6]),
               dict(out_q=tokens.transpose(1, 2)[:, :4, 1:5], out_k=tokens.transpose(1, 2)[:, 4:, 1:5]),
               dict(out_q=tokens.transpose(1, 2)[:, :4, 1:5], out_k=tokens.transpose(1, 2)[:, :2, 5:])):
        with pytest.raises(ValueError, match="CUDA"):
            hira_qk_norm_rope(**{**dict(query=q, key=k, cos=c, sin=c), **kw})


def test_shared_memory_is_found_byte_by_byte():
    gen = torch.Generator().manual_seed(0)
    buf = torch.arange(600, dtype=torch.int32)

    def pick(n):
        return int(torch.randint(n, (1,), generator=gen))
    met = 0
    for _ in range(400):
        views = []
        for _ in range(2):
            shape = [1 + pick(4) for _ in range(3)]
            stride = [pick(40), pick(12), 1 + pick(2)]
            views.append(buf.as_strided(shape, stride, pick(200)))
        a, b = views
        want = bool(set(a.flatten().tolist()) & set(b.flatten().tolist()))
        assert S.share_memory(a, b) == want == S.share_memory(b, a)
        met += want
    assert 50 < met < 350
    big, accepted = torch.arange(4000, dtype=torch.int32), 0
    for _ in range(400):         # what passes as writable has no element twice
        t = big.as_strided((1 + pick(4), 1 + pick(4), 1 + pick(4), 4), (4 * pick(40), 4 * pick(12), 4 * pick(3), 1))
        if S.writable_rows(t):
            accepted += 1
            assert len(set(t.flatten().tolist())) == t.numel()
    assert accepted > 40
    assert S.share_memory(buf.view(torch.int8)[3:4], buf[:1]) and not S.share_memory(buf[:0], buf) and not S.share_memory(buf.clone(), buf)


def test_shared_attention_refuses_an_output_that_overlaps_what_is_read():
    a = {k: _t(*s) for k, s in GOOD.items()}
    buf = _t(6, 9, 3, 64)
    lens = torch.zeros(2, dtype=torch.int32)
    for kw, match in ((dict(query=buf[:, :4, :1], out=buf[:, 1:5, :1]), "query"), (dict(tail_keys=buf[:, :2], out=buf[:, 1:5, 2:]), "tail_keys"),
                      (dict(tail_values=buf[:, 5:7], out=buf[:, 3:7, :1]), "tail_values"),
                      (dict(prefix_keys=buf.view(2, -1, 9, 64)[:, :2], out=buf[:, :4, :1]), "prefix_keys"),
                      (dict(prefix_lens=lens, out=lens.as_strided((1,), (1,)).view(torch.bfloat16)), "out must be"),
                      (dict(out=buf[:, :4, :1].as_strided((6, 4, 1, 64), (64, 64, 64, 1))), "out must be")):
        with pytest.raises(ValueError, match=match):
            hira_shared_attention(**{**a, **kw})
    for kw in (dict(out=a["query"]), dict(query=buf[:, :4, :1], out=buf[:, :4, 1:2]), dict(tail_keys=buf[:, :2], tail_values=buf[:, 2:4], out=buf[:, 4:8, 1:2])):
        with pytest.raises(ValueError, match="CUDA"):
            hira_shared_attention(**{**a, **kw})


@pytest.mark.parametrize("code,match", [(8, "does not exist"), (4, "gave up"), (1, "capacity"), (2, "capacity"), (9, "does not exist")])
def test_a_shared_prompt_reports_all_that_an_index_does(code, match):
    p = SharedPrompt(_t(1, 1, 3, 8), _t(1, 1, 3, 8), 2)
    p.check_status()
    p.status.fill_(code)
    with pytest.raises(RuntimeError, match=match):
        p.check_status()


@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_not_dropped_in_silence(grad):
    import torch.autograd.forward_ad as fw
    a = {k: _t(*s, dtype=torch.float32) for k, s in GOOD.items()}
    q, k, c = _t(2, 4, 4, 64, dtype=torch.float32), _t(2, 2, 4, 64, dtype=torch.float32), _t(2, 4, 64, dtype=torch.float32)
    with torch.set_grad_enabled(grad), fw.dual_level():
        for name, t in a.items():
            with pytest.raises(ValueError, match="forward mode"):
                hira_shared_attention(**{**a, name: fw.make_dual(t, torch.ones_like(t))})
        for kw in (dict(query=q), dict(key=k), dict(cos=c), dict(sin=c), dict(q_weight=_t(64, dtype=torch.float32)), dict(k_weight=_t(64, dtype=torch.float32))):
            for name, t in kw.items():
                with pytest.raises(ValueError, match="forward mode"):
                    hira_qk_norm_rope(**{**dict(query=q, key=k, cos=c, sin=c), name: fw.make_dual(t, torch.ones_like(t))})
        with pytest.raises(ValueError, match="CUDA"):
            hira_shared_attention(**a)
        with pytest.raises(ValueError, match="CUDA"):
            hira_qk_norm_rope(q, k, c, c)


def test_a_shared_prompt_takes_no_keys_that_would_have_to_be_differentiated():
    import torch.autograd.forward_ad as fw
    p, new = SharedPrompt(_t(1, 1, 3, 8, dtype=torch.float32), _t(1, 1, 3, 8, dtype=torch.float32), 2), _t(2, 1, 1, 8, dtype=torch.float32)
    for args in ((new.clone().requires_grad_(), new), (new, new.clone().requires_grad_())):
        with pytest.raises(ValueError, match="no backward"):
            p.append(*args)
        assert p.tail_len == 0
        with torch.no_grad():
            p.select([0, 1]).append(*args)
    with fw.dual_level(), torch.no_grad(), pytest.raises(ValueError, match="forward mode"):
        p.append(new, fw.make_dual(new, new))
    assert p.append(new, new).tail_len == 1 and not p.tail_keys.requires_grad


def test_a_shared_prompt_takes_keys_of_its_own_type_only():
    p, new = SharedPrompt(_t(1, 1, 3, 8), _t(1, 1, 3, 8), 2), _t(2, 1, 1, 8)
    for args in ((new.float(), new), (new, new.float()), (new.half(), new.half()), (new.to("meta"), new), (new, new.int())):
        with pytest.raises(ValueError, match="the tails"):
            p.append(*args)
        assert p.tail_len == 0
    assert p.append(new, new).tail_len == 1


def test_samples_that_nobody_holds_are_not_kept_track_of():
    from types import SimpleNamespace

    from hira_b200.attention.hira_attention import _samples_for
    st = S.IndexState(n_heads=2, dim=8, vdim=8, bf=8, depth=2, cap_parents=16, dtype=torch.float32, vdtype=torch.float32, device="cpu")
    st.slot2token[:] = torch.arange(128, dtype=torch.int32)
    ix = SimpleNamespace(state=st)
    held = _samples_for(ix, 16)
    for s in [32, 64] * 20:
        assert _samples_for(ix, s).shape == (2, s, 8)
    assert len(ix._tau_drawn) <= 3 and any(ref() is held for ref in ix._tau_drawn)


def test_a_wait_that_ran_out_has_a_status_bit_of_its_own():
    p = SharedPrompt(_t(1, 1, 3, 8), _t(1, 1, 3, 8), 2)
    p.status.fill_(L.HIRA_STATUS_ATTN_FAILED)
    for q in (p, p.select([0, 1, 1])):
        with pytest.raises(RuntimeError, match="HIRA_STATUS_ATTN_FAILED"):
            q.check_status()
    a = {k: _t(*s) for k, s in GOOD.items()}
    for status in (torch.zeros(1), torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32, device="meta")):
        with pytest.raises(ValueError, match="status"):
            hira_shared_attention(**a, status=status)
    with pytest.raises(ValueError, match="CUDA"):
        hira_shared_attention(**a, status=torch.zeros(1, dtype=torch.int32))
    lib, args = L.load(), _args(status=4097)
    assert lib.hira_shared_attn_workspace_bytes(C.byref(args)) == 0 and lib.hira_shared_attn(C.byref(args), None, 0, None) == L.HIRA_ERR_ARG
    args.status = 4096
    assert lib.hira_shared_attn(C.byref(args), None, 0, None) == L.HIRA_ERR_CAPACITY


def _parts(**kw):
    """Parts of an output row, from the size of the workspace (a tail that joins the parts itself has none)."""
    a = _args(**{**dict(group=1, tail_len=0), **kw})
    rows = a.n_prompts * a.n_branches * a.n_kv * a.group * a.n_q
    n, rest = divmod(L.load().hira_shared_attn_workspace_bytes(C.byref(a)), 4 * (a.vdim + 2) * rows)
    assert rest == 0
    return n


@pytest.mark.parametrize("width", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 8, 16])
@pytest.mark.parametrize("n_kv", [1, 2, 3, 8])
def test_long_prompts_of_few_heads_keep_the_device_busy(n_kv, rows, width):
    for n in (1, 64, 200, 3000, 32768, 65536, 131072, 1 << 20):
        parts = _parts(n_kv=n_kv, n_branches=rows, dim=width, vdim=width, prefix_len=n)
        # all 148 SMs have a block, or the blocks are short (2,048 keys)
        assert 1 <= parts <= 256 and (n_kv * (parts + 1) > 148 or n / parts <= 2048)
        assert _parts(n_kv=n_kv, n_branches=rows, dim=width, vdim=width, prefix_len=n, tail_len=n) <= 512


@pytest.mark.parametrize("n_kv,rows,width,resident", [
    # blocks of 8, 16, 32 and 64 rows take 73, 79, 92 and 116 KiB at 128 channels, 145 and more at 256: what 228 hold, at most three
    (8, 8, 128, 3), (8, 16, 128, 2), (8, 32, 128, 2), (8, 64, 128, 1), (1, 8, 128, 3), (1, 16, 128, 2), (3, 64, 128, 1), (8, 8, 256, 1),
    (1, 16, 256, 1), (8, 64, 256, 1), (8, 8, 64, 3), (8, 64, 64, 2),
])
def test_splits_in_fp32_are_the_blocks_that_are_resident_at_once(n_kv, rows, width, resident):
    block = 8 if rows <= 8 else 16 if rows <= 16 else 32 if rows <= 32 or width > 128 else 64
    blocks = -(-rows // block) * n_kv
    for n in (64, 1000, 32768, 100000):
        parts = _parts(dtype=L.HIRA_F32, n_kv=n_kv, n_branches=rows, dim=width, vdim=width, prefix_len=n)
        assert parts == max(1, min(resident * 148 // blocks, (-(-n // 64) + 1) // 2, 256))
