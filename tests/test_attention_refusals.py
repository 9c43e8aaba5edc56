"""The attention operators' Python functions with arguments that are not tensors, or of another number of dimensions: a
TypeError or a ValueError that names the argument, as the module says, before anything is launched.  The functions behind
the entries are called with tensors of the CPU, for which no call gets past its checks."""
from types import SimpleNamespace

import pytest
import torch


@pytest.fixture(scope="module")
def A():
    from exl3_b200 import attention

    return attention


def ints(*v):
    return torch.tensor(v, dtype=torch.int32)


@pytest.fixture
def cache():
    return SimpleNamespace(_index=-1, kv_heads=2, head_dim=64, _scratch={(3, 4): 0}, _at=0, device="cpu",
                           scratch_bytes=lambda rows, heads: 0)


q, kv = torch.zeros(3, 4, 64), torch.zeros(3, 2, 64)
h, hkv = q.half(), kv.half()
pos, offs = ints(0, 1, 2), ints(0, 3)
flat = ints(5).reshape(())

ROPE = dict(q=q, k=kv, positions=pos)
APPEND = dict(k=kv, v=kv, row_seq=pos, row_pos=pos, seq_slot=offs)
READ = dict(seq_slot=ints(0), kv_offsets=offs, total_rows=3)
ATTEND = dict(q=q, row_seq=pos, row_pos=pos, seq_slot=offs)
PROMPT = dict(q=h, k=hkv, v=hkv, q_offsets=offs, kv_offsets=offs)

NOT_TENSORS = [("qk_norm_rope", ROPE, n) for n in ("q", "k", "positions", "inv_freq", "q_weight", "k_weight", "q_out", "k_out")]
NOT_TENSORS += [("append", APPEND, n) for n in APPEND]
NOT_TENSORS += [("read", READ, n) for n in ("seq_slot", "kv_offsets", "k_out", "v_out")]
NOT_TENSORS += [("attend", ATTEND, n) for n in (*ATTEND, "out", "scratch")]
NOT_TENSORS += [("prompt_attention", PROMPT, n) for n in (*PROMPT, "out", "scratch")]


def call(A, cache, name, kw):
    fn = getattr(A, name, None)
    return fn.__wrapped__(**kw) if fn else getattr(A.Kv4Cache, name).__wrapped__(cache, **kw)


@pytest.fixture(autouse=True)
def no_launch(A, monkeypatch):
    def launch(*a):
        pytest.fail("launched")

    for name in ("_rope_call", "_append_call", "_read_call", "_attn_call", "_prompt_call"):
        monkeypatch.setattr(A, name, launch)
    monkeypatch.setattr(A, "_stream", lambda index: 0)


@pytest.mark.parametrize("name,args,bad", NOT_TENSORS)
@pytest.mark.parametrize("value", [[1, 2, 3], 7, "x"])
def test_what_is_not_a_tensor_is_named(A, cache, name, args, bad, value):
    with pytest.raises(TypeError, match=bad):
        call(A, cache, name, {**args, bad: value})


@pytest.mark.parametrize("name,args,bad", [(n, a, b) for n, a, b in NOT_TENSORS
                                           if b in ("q", "k", "v", "positions", "row_seq", "row_pos", "seq_slot", "q_offsets")])
def test_a_missing_tensor_is_named(A, cache, name, args, bad):
    if bad == "k" and name == "qk_norm_rope":
        return  # no keys is a call
    with pytest.raises(TypeError, match=bad):
        call(A, cache, name, {**args, bad: None})


@pytest.mark.parametrize("name,args,bad", [
    ("qk_norm_rope", ROPE, "inv_freq"), ("qk_norm_rope", ROPE, "positions"), ("append", APPEND, "seq_slot"), ("append", APPEND, "row_pos"),
    ("read", READ, "seq_slot"), ("read", READ, "kv_offsets"), ("attend", ATTEND, "seq_slot"), ("prompt_attention", PROMPT, "q_offsets"),
    ("prompt_attention", PROMPT, "kv_offsets"), ("prompt_attention", {**PROMPT, "kv_offsets": None, "kv_end": offs}, "kv_begin")])
def test_a_scalar_tensor_is_refused(A, cache, name, args, bad):
    with pytest.raises(ValueError, match=bad):
        call(A, cache, name, {**args, bad: flat})


def test_numbers_that_are_none(A, cache):
    with pytest.raises(ValueError, match="total_rows"):
        call(A, cache, "read", {**READ, "total_rows": -1})
    pack = A._call(0, "if")  # the conversion of a call's arguments, before its entry is reached
    for bad in (("x", 1.0), (1, "x"), (1, None), (1 << 70, 1.0), (1, 10 ** 400)):
        with pytest.raises(TypeError, match="number"):
            pack(*bad)


@pytest.mark.parametrize("name", ["qk_norm_rope", "prompt_attention"])
@pytest.mark.parametrize("first", [[1, 2], 3.0, "q"])
def test_a_first_argument_that_is_no_tensor(A, name, first):
    with pytest.raises(TypeError, match="takes tensors"):
        getattr(A, name)(first, q, q, pos)
