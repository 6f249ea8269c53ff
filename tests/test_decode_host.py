"""Token decoding, the parts that need no GPU: the operators' registration and shapes, the ctypes
mirrors, refusals before any device work, and the cache's page bookkeeping (on CPU tensors)."""

import ctypes as C

import pytest
import torch

import rldx_b200.torch_ops  # noqa: F401  (registers torch.ops.b200msat)
from rldx_b200 import _lib, ops
from rldx_b200.decoder import B200KV4Cache

BF, I32 = torch.bfloat16, torch.int32


def test_struct_sizes():
    assert C.sizeof(_lib.Kv4Cache) == 5 * 8 + 6 * 4
    assert C.sizeof(_lib.Kv4AttentionDesc) == 3 * 8 + 8 * 4


def test_fake_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        cache = torch.empty(9, 2, 2, 40 * 128, dtype=torch.uint8)
        table, lengths, cu = torch.empty(3, 4, dtype=I32), torch.empty(3, dtype=I32), torch.empty(4, dtype=I32)
        t = torch.empty(50, 128)
        q = torch.ops.b200msat.qkv_rope_append(torch.empty(7, 20 * 128, dtype=BF), torch.empty(128, dtype=BF),
                                               torch.empty(128, dtype=BF), t, t, torch.empty(7, dtype=I32), cache, table,
                                               lengths, cu, 16)
        assert q.shape == (7, 16, 128) and q.dtype == BF
        k, v = torch.ops.b200msat.kv4_read(cache, table, lengths, cu, 7)
        assert k.shape == v.shape == (7, 2, 128) and k.dtype == BF
        assert torch.ops.b200msat.kv4_attention(q, cache, table, lengths, cu, 3, 100).shape == q.shape
        token, logprob, kept = torch.ops.b200msat.sample(torch.empty(5, 99, dtype=BF), torch.empty(5))
        assert (token.dtype, logprob.dtype, kept.dtype) == (torch.int64, torch.float32, I32) and token.shape == (5,)


def test_cpu_tensors_are_refused():
    cache = ops.kv4_cache(4, 2, 64, 32, device="cpu")
    assert cache.shape == (4, 2, 1, 2560)
    table, lengths, cu = torch.zeros(1, 1, dtype=I32), torch.ones(1, dtype=I32), torch.tensor([0, 1], dtype=I32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv4_attention(torch.zeros(1, 4, 64, dtype=BF), cache, table, lengths, cu, max_new=1, max_len=1)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv4_read(cache, table, lengths, cu, tokens=1)
    with pytest.raises(ValueError, match="CUDA"):
        ops.sample(torch.zeros(2, 10), torch.zeros(2))
    one = torch.ones(64, dtype=BF)
    with pytest.raises(ValueError, match="CUDA"):
        ops.qkv_rope_append(torch.zeros(1, 8 * 64, dtype=BF), one, one, torch.ones(1, 64), torch.zeros(1, 64),
                            torch.zeros(1, dtype=I32), cache, table, lengths, cu, q_heads=4)


def test_library_refuses_without_a_device_or_with_nulls(lib):
    n = C.c_uint64(7)
    assert lib.rldx_kv4_attention_workspace_size(None, None, C.byref(n)) == _lib.RLDX_ERR_ARG and n.value == 0
    assert lib.rldx_kv4_attention_workspace_size(None, None, None) == _lib.RLDX_ERR_ARG
    c = _lib.Kv4Cache(256, 256, 256, 256, 10, 64, 2, 128, 4, 4, 1)
    a = _lib.Kv4AttentionDesc(None, None, 0, 1, 16, 1, 200, 0, 0, 0.1)
    assert lib.rldx_kv4_attention_workspace_size(C.byref(c), C.byref(a), C.byref(n)) == _lib.RLDX_OK
    for field, value, rc in (("head_dim", 96, _lib.RLDX_ERR_UNSUPPORTED), ("page_size", 48, _lib.RLDX_ERR_ARG),
                             ("kv_heads", 3, _lib.RLDX_ERR_ARG), ("table_ld", 3, _lib.RLDX_ERR_ARG), ("pages", 0, _lib.RLDX_ERR_ARG),
                             ("pages", 1 << 30, _lib.RLDX_ERR_UNSUPPORTED), ("data", 264, _lib.RLDX_ERR_ARG), ("seqs", 0, _lib.RLDX_ERR_ARG)):
        bad = _lib.Kv4Cache.from_buffer_copy(c)
        setattr(bad, field, value)
        assert lib.rldx_kv4_attention_workspace_size(C.byref(bad), C.byref(a), C.byref(n)) == rc, field


def test_cache_pages():
    c = B200KV4Cache(2, 1, 64, seqs=3, max_tokens=320, page_size=32, device="cpu")
    assert len(c.pools) == 2 and c.pools[0].shape == (13, 1, 1, 2560)
    c.extend([33, 0, 64])
    assert c.tokens == [33, 0, 64] and c.lengths.tolist() == [33, 0, 64]
    held = [c.table[s][c.table[s] >= 0].tolist() for s in range(3)]
    assert [len(h) for h in held] == [2, 0, 2] and len(set(sum(held, []))) == 4
    c.extend([31, 1, 1])  # the first sequence's second page has room
    again = [c.table[s][c.table[s] >= 0].tolist() for s in range(3)]
    assert again[0] == held[0] and len(again[1]) == 1 and again[2][:2] == held[2] and len(again[2]) == 3
    free = c.free_tokens
    c.release(2)
    assert c.free_tokens == free + 96 and c.lengths.tolist() == [64, 1, 0] and int(c.table[2].max()) == -1
    with pytest.raises(RuntimeError, match="free pages"):
        c.extend([10000, 0, 0])
    assert c.tokens == [64, 1, 0]
    with pytest.raises(ValueError):
        c.extend([1, 1])
    with pytest.raises(ValueError):
        c.extend([-1, 0, 0])
