"""Argument checks of the paged serving operators that need no GPU."""

import ctypes

import pytest
import torch

import hf_attention_normalizers_b200 as H
from hf_attention_normalizers_b200 import _native as N
from hf_attention_normalizers_b200 import serving


def _args(**kw):
    a = dict(query=torch.zeros(3, 4, 16), key_cache=torch.zeros(64, 2, 16), value_cache=torch.zeros(64, 2, 16),
             block_table=torch.zeros(2, 2, dtype=torch.int32), cu_seqlens_q=torch.tensor([0, 1, 3], dtype=torch.int32),
             sequence_lengths=torch.tensor([5, 9], dtype=torch.int32), block_size=16)
    a.update(kw)
    return a


def test_serving_is_reached_through_the_package():
    assert H.serving is serving and all(callable(getattr(serving, n)) for n in serving.__all__)


@pytest.mark.parametrize("kw,msg", [
    (dict(), "requires CUDA tensors"),
    (dict(key_cache=torch.zeros(64, 32)), "must have matching"),
    (dict(value_cache=torch.zeros(64, 2, 8)), "must have matching"),
    (dict(value_cache=torch.zeros(64, 2, 16).half()), "one dtype"),
    (dict(value_cache=torch.zeros(64, 16, 2).transpose(1, 2)), "unit innermost stride"),
])
def test_cache_checks(kw, msg):
    with pytest.raises(ValueError, match=msg):
        serving.paged_chunk_attention(**_args(**kw))
    a = _args(**kw)
    with pytest.raises(ValueError, match=msg):
        serving.paged_append(torch.zeros(3, 2, 16), torch.zeros(3, 2, 16), a["key_cache"], a["value_cache"],
                             a["block_table"], a["cu_seqlens_q"], a["sequence_lengths"], 16)
    with pytest.raises(ValueError, match=msg):
        serving.paged_evict(a["key_cache"], a["value_cache"], torch.zeros(2, 64), a["block_table"], a["sequence_lengths"],
                            16, 4)


def _desc(**kw):
    d = dict(dtype=N.BFLOAT16, normalizer=N.SOFTMAX1, batch=2, heads_q=4, heads_kv=2, head_dim=64, total_q=3, max_len_q=2,
             page_size=16, max_blocks=2, max_len_k=32, num_cache_tokens=64, block_table=1, cu_seqlens_q=1, seq_lens=1,
             scale=0.1, causal=1)
    d.update(kw)
    return N.ChunkDesc(**d)


@pytest.mark.parametrize("kw,msg", [
    (dict(normalizer=5), "unknown normalizer"),
    (dict(dtype=5), "unknown dtype"),
    (dict(heads_q=5), "divisible"),
    (dict(head_dim=257), "head_dim"),
    (dict(batch=70000), "batch larger"),
    (dict(page_size=0), "block_size"),
    (dict(max_len_k=33), "enough blocks"),
    (dict(block_table=None), "required"),
    (dict(cu_seqlens_q=None), "cu_seqlens_q"),
    (dict(total_q=-1), "negative"),
    (dict(total_q=2 ** 30), "rows in one call"),
    (dict(num_cache_tokens=2 ** 31), "cache slots"),
])
def test_requests_are_refused_on_the_host(kw, msg):
    lib, t = N.lib(), N.HfanTensor(None, 0, 0, 0)
    one = ctypes.c_void_p(1)
    assert lib.hfan_paged_chunk_fwd(ctypes.byref(_desc(**kw)), t, t, t, t, one, None, 0, None, 0, None) == 1
    assert msg in lib.hfan_last_error().decode()
    assert lib.hfan_paged_append(ctypes.byref(_desc(**kw)), t, t, t, t, None, 0, None) == 1
    assert lib.hfan_paged_chunk_workspace_bytes(ctypes.byref(_desc(**kw)), 0) == -1


@pytest.mark.parametrize("budget,recent,ld,msg", [(0, 0, 64, "budget"), (4, -1, 64, "recent"), (4, 0, 63, "every cache slot")])
def test_evict_requests_are_refused_on_the_host(budget, recent, ld, msg):
    lib, t, one = N.lib(), N.HfanTensor(None, 0, 0, 0), ctypes.c_void_p(1)
    assert lib.hfan_paged_evict(ctypes.byref(_desc(cu_seqlens_q=None)), t, t, one, ld, budget, recent, one, one, None) == 1
    assert msg in lib.hfan_last_error().decode()


def test_workspace_holds_each_score_once():
    """Kept scores of 8-token chunks: four bytes a (row, key)."""
    lib = N.lib()
    d = _desc(batch=8, heads_q=8, heads_kv=2, total_q=64, max_len_q=8, max_blocks=512, max_len_k=8192)
    size = [lib.hfan_paged_chunk_workspace_bytes(ctypes.byref(d), w) for w in (0, 1)]
    assert 0 < size[0] and size[1] - size[0] == 64 * 8 * 8192 * 4


@pytest.mark.parametrize("grad", [False, True])
def test_fake_tensors(grad):
    """Outside torch.compile: shapes come from the custom ops, nothing is launched."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode(), torch.set_grad_enabled(grad):
        def make(*shape, dtype=torch.bfloat16):
            return torch.empty(*shape, dtype=dtype, device="cuda")

        kc, vc, w, table = make(64, 2, 64), make(64, 2, 64), make(2, 64, dtype=torch.float32), make(2, 2, dtype=torch.int32)
        cu, lens = make(3, dtype=torch.int32), make(2, dtype=torch.int32)
        assert serving.paged_append(make(3, 2, 64), make(3, 2, 64), kc, vc, table, cu, lens, 16, key_weights=w) is None
        out = serving.paged_chunk_attention(make(3, 4, 64), kc, vc, table, cu, lens, 16, key_weights=w)
        assert out.shape == (3, 4, 64) and out.dtype is torch.bfloat16 and out.device.type == "cuda"
        lens, kept = serving.paged_evict(kc, vc, w, table, lens, 16, 10)
        assert lens.shape == (2,) and kept.shape == (2, 2, 10) and kept.dtype is torch.int32


def test_cache_on_the_device_of_its_pages():
    """A cache made for "cuda" stays with the device that was current then."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        cache = serving.PagedServingCache(1, 2, 4, 16, 1, 64)
        assert cache._device == cache.layers[0].device and cache._device.index is not None


def test_release_ends_one_sequence():
    """Its pages go to others, and its place takes a new text."""
    cache = serving.PagedServingCache(1, 3, 6, 16, 1, 64, device="cpu")
    cache.step([40, 16, 20])
    with pytest.raises(ValueError, match="no room"):
        cache.step([0, 16, 0])
    cache.release(0)
    assert cache.lengths == [0, 16, 20]
    step = cache.step([5, 16, 13])
    assert cache.lengths == [5, 32, 33] and step.lengths.tolist() == [5, 32, 33]
    used = [p for b, n in enumerate((1, 2, 3)) for p in step.block_table[b, :n].tolist()]
    assert sorted(used) == list(range(6))
    cache.release(1)
    cache.release(1)  # nothing left to free
    assert cache.step([0, 0, 31]).max_seqlen_k == 64
    for b in (3, -1):
        with pytest.raises(ValueError, match="no sequence"):
            cache.release(b)
