"""Refusals of the serving operators without a GPU: the C ABI checks its arguments before any CUDA
call (the pointers here are never read), the Python layer refuses what has no CUDA path. The plain
page model the GPU tests follow is checked against its own definition."""
import ctypes

import pytest
import torch

from respect_b200 import _lib
from tests.serving_reference import Pages

OK, INVALID, UNSUPPORTED, CAPACITY, WORKSPACE = 0, 1, 2, 3, 6


def prompt_args(**kw):
    a = _lib.PromptArgs(_lib.RB_BF16, 1, 4, 8, 2, 128, 0x100000, 1024, 128, 0x200000, 256, 128, 0x300000, 256, 128,
                        0x400000, 0x500000, 1024, 128, 0.1, 0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,status", [
    (dict(q=None), INVALID), (dict(cu=None), INVALID), (dict(out=None), INVALID), (dict(B=-1), INVALID),
    (dict(T=-1), INVALID), (dict(H=0), INVALID), (dict(HK=0), INVALID), (dict(sm_scale=float("nan")), INVALID),
    (dict(D=64), UNSUPPORTED), (dict(HK=3), UNSUPPORTED), (dict(H=65, HK=1), UNSUPPORTED),
    (dict(dtype=_lib.RB_I32), UNSUPPORTED), (dict(q=0x100008), UNSUPPORTED), (dict(skt=252), UNSUPPORTED),
    (dict(svh=4), UNSUPPORTED), (dict(sot=-1024), UNSUPPORTED), (dict(T=0), OK)])
def test_prompt_refusals(change, status):
    assert _lib.lib().rb_prompt_attn(ctypes.byref(prompt_args(**change)), None) == status


def paged_args(**kw):
    a = _lib.PagedArgs(_lib.RB_BF16, 2, 8, 2, 128, 0x100000, 1024, 128, 0x200000, 4096, 2048, 128, 0x300000, 4096, 2048,
                       128, 10, 16, 0x400000, 40, 40, 2, 0x500000, None, 0, 0, 0x600000, 1024, 128, 0.1)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,status", [
    (dict(q=None), INVALID), (dict(k=None), INVALID), (dict(table=None), INVALID), (dict(lengths=None), INVALID),
    (dict(page_size=0), INVALID), (dict(ahead=-1), INVALID), (dict(ld_table=39), INVALID), (dict(width=-1), INVALID),
    (dict(sm_scale=float("nan")), INVALID), (dict(D=64), UNSUPPORTED), (dict(HK=3), UNSUPPORTED),
    (dict(dtype=_lib.RB_U8), UNSUPPORTED), (dict(skp=4100), UNSUPPORTED), (dict(v=0x300002), UNSUPPORTED),
    (dict(B=70000), CAPACITY), (dict(width=1 << 28, ld_table=1 << 28), CAPACITY), (dict(B=0), OK),
    (dict(), WORKSPACE)])      # 640 tokens take several chunks: scratch is needed
def test_paged_refusals(change, status):
    assert _lib.lib().rb_paged_attn(ctypes.byref(paged_args(**change)), None, 0, None) == status


def test_paged_workspace_follows_the_bound_on_the_length():
    need = _lib.lib().rb_paged_attn_workspace
    assert need(ctypes.byref(paged_args(max_length=60))) == 0
    assert need(ctypes.byref(paged_args())) > 0
    assert need(ctypes.byref(paged_args(D=64))) == 0


def pages_args(**kw):
    a = _lib.KVPages(0x100000, 2, 10, 2, 16, 128, 2, 4, 10, 0x200000, 0x300000, 0x400000, 0x500000, 0x600000)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_page_operations_refuse():
    lib = _lib.lib()
    p = 0x700000
    for change, status in ((dict(store=None), INVALID), (dict(status=None), INVALID), (dict(pages=0), INVALID),
                           (dict(page_size=0), INVALID), (dict(elem_bytes=1), UNSUPPORTED), (dict(head_dim=3), UNSUPPORTED),
                           (dict(store=0x100008), UNSUPPORTED), (dict(max_pages=1 << 28), CAPACITY),
                           (dict(pages=(1 << 20) + 1), CAPACITY), (dict(layers=20000), CAPACITY)):
        c = ctypes.byref(pages_args(**change))
        assert lib.rb_kv_pages_workspace(c) == 0
        assert lib.rb_kv_pages_commit(c, p, p, 1, None) == status
        assert lib.rb_kv_pages_truncate(c, p, p, 1, None) == status
    c = ctypes.byref(pages_args())
    ws = lib.rb_kv_pages_workspace(c)
    assert ws > 0
    assert lib.rb_kv_pages_reserve(c, p, p, 1, p, ws - 1, None) == WORKSPACE
    assert lib.rb_kv_pages_fork(c, p, p, 1, None, ws, None) == WORKSPACE
    assert lib.rb_kv_pages_compact(c, p, p, 4, 5, p, 1, p, ws, None) == INVALID     # rows closer than they are wide
    for n, status in ((-1, INVALID), (1025, CAPACITY), (0, OK)):
        assert lib.rb_kv_pages_reserve(c, p, p, n, p, ws, None) == status
        assert lib.rb_kv_pages_commit(c, p, p, n, None) == status
        assert lib.rb_kv_pages_fork(c, p, p, n, p, ws, None) == status
        assert lib.rb_kv_pages_truncate(c, p, None, n, None) == status
        assert lib.rb_kv_pages_compact(c, p, p, 4, 4, p, n, p, ws, None) == status
    x = _lib.KVTokens(p, p, 0, 256, 128, 0, 256, 128, 0, 1, 4)
    for change, status in ((dict(layer0=2), INVALID), (dict(layers=3), INVALID), (dict(tokens=-1), INVALID),
                           (dict(skt=252), UNSUPPORTED), (dict(v=p + 2), UNSUPPORTED), (dict(k=None), INVALID),
                           (dict(tokens=0), OK)):
        y = _lib.KVTokens.from_buffer_copy(x)
        for k, v in change.items():
            setattr(y, k, v)
        assert lib.rb_kv_pages_write(c, ctypes.byref(y), p, None, 1, None) == status


def test_token_logprobs_refusals():
    lib = _lib.lib()
    p = 0x100000
    ws = lib.rb_token_logprobs_workspace(4, 1000, 5)

    def call(dtype=_lib.RB_F32, ld=1000, M=4, V=1000, tokens=p, off=0, size=0, top=5, ids=p, w=p, n=ws):
        return lib.rb_token_logprobs(p, dtype, ld, M, V, tokens, off, size, top, p, p, p, ids, w, n, None)

    assert call(ld=999) == INVALID and call(M=-1) == INVALID and call(V=0) == INVALID and call(off=-1) == INVALID
    assert call(size=-1) == INVALID and call(tokens=None) == INVALID and call(ids=None) == INVALID
    assert call(V=4, ld=4) == INVALID                     # more alternatives than entries
    assert call(top=33) == CAPACITY
    assert call(dtype=_lib.RB_I64) == UNSUPPORTED
    assert call(w=None) == WORKSPACE and call(n=ws - 1) == WORKSPACE
    assert call(M=0) == OK


def test_python_layer_refuses_cpu_tensors_and_bad_shapes():
    from respect_b200.decoding.acceptance import token_logprobs
    from respect_b200.decoding.kv_pages import PagedKVCache
    from respect_b200.kernels import paged_attention, prompt_attention
    q, kv = torch.zeros(4, 8, 128), torch.zeros(4, 2, 128)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError):
        prompt_attention(q, kv, kv, cu)                   # no CPU path
    with pytest.raises(ValueError):
        prompt_attention(q, kv[:3], kv[:3], cu)
    with pytest.raises(ValueError):
        prompt_attention(q[:, :7], kv, kv, cu)
    with pytest.raises(TypeError):
        prompt_attention(q.half(), kv.half(), kv.half(), cu)
    with pytest.raises(TypeError):
        prompt_attention(q, kv, kv, cu.long())
    with pytest.raises(TypeError):
        prompt_attention(q, kv.bfloat16(), kv.bfloat16(), cu)
    with pytest.raises(ValueError):
        prompt_attention(q, kv, kv, cu, out=torch.zeros(4, 8, 64))
    pages, table, n = torch.zeros(3, 2, 16, 128), torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError):
        paged_attention(q, pages, pages, table, n)        # no CPU path
    with pytest.raises(ValueError):
        paged_attention(q, pages, pages, table[:3], n[:3])
    with pytest.raises(ValueError):
        paged_attention(q, pages, pages, table, n[:3])
    with pytest.raises(ValueError):
        paged_attention(q, pages, pages, table, n, ahead=-1)
    with pytest.raises(ValueError):
        paged_attention(q, pages, pages, table, n, max_length=0)
    with pytest.raises(ValueError):
        PagedKVCache(1, 1, 4, 16, 2, device="cpu")
    with pytest.raises(ValueError):
        PagedKVCache(1, 1, 0, 16, 2, device="cpu")
    x, t = torch.zeros(2, 10), torch.zeros(2, dtype=torch.int64)
    for bad in (dict(logits=x, tokens=t), dict(logits=x, tokens=t[:1]), dict(logits=x, tokens=t.int()),
                dict(logits=x, tokens=t, top=11), dict(logits=x, tokens=t, top=-1), dict(logits=x, tokens=t, offset=-1)):
        with pytest.raises(ValueError):
            token_logprobs(**bad)
    with pytest.raises(TypeError):
        token_logprobs(x.half(), t)


def test_plain_page_model():
    m = Pages(pages=6, page_size=4, max_seqs=3, max_pages=6)
    assert m.reserve([0], [6]) and m.rows[0] == [0, 1]
    m.write(0, list("abcdef"))
    m.commit(0, 6)
    m.fork(0, 1)
    m.fork(0, 2)
    assert m.refs[:3] == [3, 3, 0]
    assert m.reserve([1, 2, 0], [1, 1, 1])     # the last holder keeps the shared page
    assert m.rows == [[0, 1], [0, 2], [0, 3]] and m.refs == [3, 1, 1, 1, 0, 0]
    m.write(1, ["x"])
    m.commit(1, 1)
    assert "".join(m.tokens(1)) == "abcdefx" and "".join(m.tokens(0)) == "abcdef"
    assert not m.reserve([0, 1], [12, 4]) and m.refs == [3, 1, 1, 1, 0, 0]
    assert m.reserve([1], [5])
    m.write(1, list("12345"))
    m.compact(1, [1, 3])
    assert "".join(m.tokens(1)) == "abcdefx24"
    m.truncate(1, 0)
    assert m.refs == [2, 1, 0, 1, 0, 0]


def test_packed_arguments_have_the_layout_of_the_mirrors():
    """The bytes the Python layer fills equal the ctypes mirrors of the C structures, field by field."""
    prompt = list(range(1, 20)) + [0.5, 1]
    paged = list(range(1, 30)) + [0.5]
    for pack, mirror, values in ((_lib.pack_prompt_args, _lib.PromptArgs, prompt),
                                 (_lib.pack_paged_args, _lib.PagedArgs, paged)):
        packed = pack(*values)
        want = bytes(mirror(*values))
        assert want.startswith(packed) and not any(want[len(packed):])
