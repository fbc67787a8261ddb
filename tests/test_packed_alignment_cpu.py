"""Alignment that the kernels' widest accesses need, checked by the C ABI before any launch (no GPU: nothing can be launched)."""
import pytest
import torch

from test_packed_cpu import BIG, _bwd, _extend, _fwd, _prefix, _store

CALLS = {"es_packed_attn_fwd": (_fwd, ("o", "rest", "ws")), "es_packed_attn_bwd": (_bwd, ("dq", "dk", "dv", "ws")), "es_prefix_attn": (_prefix, ("ws",))}
WIDE = [(name, arg) for name, (_, args) in CALLS.items() for arg in args]


@pytest.mark.skipif(torch.cuda.is_available(), reason="the pointers are made up: without a GPU no call can reach a kernel with them")
@pytest.mark.parametrize("name,arg", WIDE)
@pytest.mark.parametrize("off", [4, 8, 16])
def test_what_is_stored_32_bytes_at_once(name, arg, off):
    """All of these receive 32-byte stores: at 16 mod 32 a store would be misaligned on the device."""
    from self_trainable_or_free_attn_b200 import _native
    fn, make, before = getattr(_native.load(), name), CALLS[name][0], _native.launch_count()
    assert fn(*make(**{arg: 20 * BIG + 32}).values()) < -1, "stopped by nothing but the missing GPU"
    assert fn(*make(**{arg: 20 * BIG + off}).values()) == -1
    assert name in _native.last_error() and "aligned" in _native.last_error() and _native.launch_count() == before
    if name == "es_prefix_attn":                             # a prefix with more rows than its smallest kernel takes: the parts lie at the workspace's start
        assert fn(*make(B=70, ws=20 * BIG + off).values()) == -1


WORDS = {"es_packed_attn_fwd": (_fwd, ("lse", "cu_q", "cu_k")), "es_packed_attn_bwd": (_bwd, ("lse", "cu_q", "cu_k")),
         "es_prefix_attn": (_prefix, ("lse", "pages", "table", "lengths")), "es_store_kv": (_store, ("slots",)),
         "es_extend_tables": (_extend, ("lengths", "new", "table", "free", "slots", "pos", "cu", "out", "taken"))}


@pytest.mark.skipif(torch.cuda.is_available(), reason="the pointers are made up: without a GPU no call can reach a kernel with them")
@pytest.mark.parametrize("name,arg", [(name, arg) for name, (_, args) in WORDS.items() for arg in args])
def test_words(name, arg):
    from self_trainable_or_free_attn_b200 import _native
    fn, make = getattr(_native.load(), name), WORDS[name][0]
    assert fn(*make(**{arg: 20 * BIG + 4}).values()) < -1, "stopped by nothing but the missing GPU"
    assert fn(*make(**{arg: 20 * BIG + 2}).values()) == -1 and name in _native.last_error() and "aligned" in _native.last_error()
