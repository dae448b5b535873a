"""The paged cache's refusals, without a GPU: the C entry points reject bad arguments before any launch, the Python
functions refuse CPU tensors and mismatched shapes and types, the cache's bookkeeping refuses bad rows."""
import ctypes

import pytest
import torch

from smlm_b200 import _lib as L
from smlm_b200 import paged

P = ctypes.c_void_p(0x1000)      # never dereferenced: the checks fail before any launch
OK_STRIDES = (ctypes.c_int64 * 6)(1024, 512, 64, 1024, 512, 64)


def attention(dtype=L.BF16, strides=OK_STRIDES, q=P, k=P, batch=2, hq=4, hkv=2, d=64, pages=8, page=16, blocks=4,
              stride=4, window=0, sinks=0, ws=P, nbytes=1 << 30):
    return L.lib().smlm_paged_attention(q, k, P, dtype, strides, P, stride, P, batch, hq, hkv, d, pages, page, blocks,
                                        0.125, window, sinks, P, None, ws, nbytes, None, None)


@pytest.mark.parametrize("args,text", [
    ({"dtype": L.Q4}, b"dtype"), ({"hq": 5}, b"heads"), ({"hkv": 0}, b"heads"), ({"d": 24}, b"head dimension"),
    ({"d": 272}, b"head dimension"), ({"page": 24}, b"page_size"), ({"page": 8192}, b"page_size"),
    ({"pages": 0}, b"pages"), ({"stride": 3}, b"stride"), ({"batch": 65536}, b"batch"), ({"batch": -1}, b"batch"),
    ({"window": -1}, b"window"), ({"sinks": -1}, b"sinks"), ({"k": ctypes.c_void_p(0x1008)}, b"aligned"),
    ({"q": ctypes.c_void_p(0x1002)}, b"aligned"), ({"q": None}, b"aligned"), ({"k": None}, b"null"),
    ({"strides": (ctypes.c_int64 * 6)(1024, 512, 60, 1024, 512, 64)}, b"multiples"),
    ({"strides": (ctypes.c_int64 * 6)(1 << 33, 512, 64, 1024, 512, 64)}, b"GiB")])
def test_attention_refusals(args, text):
    assert attention(**args) == L.ERR_INVALID
    assert text in L.lib().smlm_last_error()


def test_workspaces():
    roomy = {"blocks": 60000, "stride": 60000}       # so much that it is not one launch without scratch
    assert attention(nbytes=16, **roomy) == L.ERR_WORKSPACE and attention(ws=None, **roomy) == L.ERR_WORKSPACE
    lib = L.lib()
    assert lib.smlm_paged_attention_workspace(4, 8, 2, 64, L.BF16, 16, 60000, 0, 0) > 0
    assert lib.smlm_paged_attention_workspace(4, 8, 3, 64, L.BF16, 16, 60000, 0, 0) == 0      # refused arguments
    assert lib.smlm_pages_extend(P, 4, 4, 4, P, P, 8, 16, P, 2, 1, P, 8, None, None) == L.ERR_WORKSPACE
    assert lib.smlm_pages_fork(P, 2, 2, 128, P, 4, 4, 4, P, P, 8, 16, P, P, 2, P, 8, None, None) == L.ERR_WORKSPACE
    assert lib.smlm_pages_compact(P, 2, 2, 128, P, 4, 4, 4, P, 8, 16, P, 8, None, None) == L.ERR_WORKSPACE
    # nothing to do launches nothing
    assert attention(batch=0) == L.OK
    assert lib.smlm_pages_free(P, 4, 4, 4, P, P, 8, P, 0, None, None) == L.OK


def test_append_and_page_refusals():
    lib = L.lib()

    def append(tokens=3, hq=4, d=64, cos=P, sin=P, positions=9, qkv=P):
        return lib.smlm_paged_append(qkv, P, P, L.BF16, OK_STRIDES, P, 4, P, 2, tokens, hq, 2, d, 8, 16, 4, cos, sin,
                                     positions, P, None, None)
    for args, text in [({"cos": None}, b"together"), ({"positions": 0}, b"together"), ({"tokens": -1}, b"tokens"),
                       ({"qkv": ctypes.c_void_p(0x1004)}, b"aligned"), ({"cos": ctypes.c_void_p(0x1004)}, b"aligned"),
                       ({"hq": 4096, "d": 256}, b"2^20")]:
        assert append(**args) == L.ERR_INVALID and text in lib.smlm_last_error(), args
    assert append(tokens=0) == L.OK
    assert lib.smlm_pages_free(None, 4, 4, 4, P, P, 8, P, 2, None, None) == L.ERR_INVALID
    assert lib.smlm_pages_trim(P, 4, 4, 4, P, P, 8, 16, P, 2, 0, 0, None, None) == L.ERR_INVALID
    assert b"window" in lib.smlm_last_error()
    assert lib.smlm_pages_extend(P, 4, 4, 4, P, P, 8, 12, P, 2, 1, P, 1 << 20, None, None) == L.ERR_INVALID
    assert lib.smlm_pages_extend(P, 4, 4, 4, P, P, 8, 16, P, 2, 65, P, 1 << 20, None, None) == L.ERR_INVALID
    assert lib.smlm_pages_fork(P, 2, 2, 120, P, 4, 4, 4, P, P, 8, 16, P, P, 2, P, 1 << 20, None, None) == L.ERR_INVALID
    assert b"multiple of 16" in lib.smlm_last_error()
    assert lib.smlm_pages_compact(ctypes.c_void_p(0x1008), 2, 2, 128, P, 4, 4, 4, P, 8, 16, P, 1 << 20, None,
                                  None) == L.ERR_INVALID


def tensors(dtype=torch.bfloat16):
    q, k = torch.zeros(2, 4, 64, dtype=dtype), torch.zeros(8, 2, 16, 64, dtype=dtype)
    return q, k, k.clone(), torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)


def test_python_refusals():
    q, k, v, table, lengths = tensors()
    with pytest.raises(ValueError, match="CUDA"):
        paged.paged_attention(q, k, v, table, lengths)
    with pytest.raises(ValueError, match="CUDA"):
        paged.paged_append(torch.zeros(2, 1, 8 * 64, dtype=q.dtype), k, v, table, lengths)
    with pytest.raises(ValueError, match="one type"):
        paged.paged_attention(q.float(), k, v, table, lengths)
    with pytest.raises(ValueError, match="unsupported type"):
        paged.paged_attention(q.double(), k.double(), v.double(), table, lengths)
    with pytest.raises(ValueError, match="int32"):
        paged.paged_attention(q, k, v, table.long(), lengths)
    with pytest.raises(ValueError, match="lengths"):
        paged.paged_attention(q, k, v, table, lengths[:1])
    with pytest.raises(ValueError, match="page_size"):
        paged.paged_attention(q, k, v[:, :, :8], table, lengths)
    with pytest.raises(ValueError, match="contiguous"):
        paged.paged_attention(q, k.transpose(2, 3), v.transpose(2, 3), table, lengths)
    with pytest.raises(ValueError, match="sequences"):
        paged.paged_attention(q[0], k, v, table, lengths)
    ref, rows = torch.zeros(8, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    pool = torch.zeros(1, 2, 8, 2, 16, 64)
    for call in (lambda: paged.pages_free(table, lengths, ref, rows),
                 lambda: paged.pages_trim(table, lengths, ref, rows, 16, 4),
                 lambda: paged.pages_extend(table, lengths, ref, rows, 1, 16),
                 lambda: paged.pages_fork(pool, table, lengths, ref, rows, rows),
                 lambda: paged.pages_compact(pool, table, ref)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="int32"):
        paged.pages_free(table, lengths, ref, rows.long())


@pytest.mark.parametrize("args,text", [({"page_size": 12}, "power of two"), ({"head_dim": 40}, "multiple of 16"),
                                       ({"dtype": torch.float64}, "unsupported"), ({"device": "cpu"}, "CUDA")])
def test_cache_refusals(args, text):
    kw = dict({"n_layers": 1, "n_pages": 4, "page_size": 16, "n_kv_heads": 2, "head_dim": 64, "max_seqs": 2,
               "max_len": 64}, **args)
    with pytest.raises(ValueError, match=text):
        paged.PagedKVCache(**kw)
