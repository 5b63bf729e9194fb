"""Refusals of the paged-cache operators that need no GPU: the C entry points
check their arguments before any launch, the Python calls before any C call."""
import pytest
import torch

PTR = 1 << 20  # an aligned address that no refused call reaches


def _append(lib, **kw):
    a = dict(qkv=PTR, qn=PTR, kn=PTR, cos=PTR, sin=PTR, rows=64, eps=1e-6, k=PTR, v=PTR, pages=4, page=16, table=PTR,
             width=4, q_start=PTR, kv=PTR, seqs=1, tokens=1, first=0, hq=16, hkv=8, out=PTR, status=PTR, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.qb_rope_paged_append(*a.values())


def _attention(lib, **kw):
    a = dict(q=PTR, k=PTR, v=PTR, pages=4, page=16, table=PTR, width=4, q_start=PTR, kv=PTR, seqs=1, tokens=1, max_q=1,
             hq=16, hkv=8, window=0, sinks=0, out=PTR, ws=PTR, ws_bytes=1 << 40, status=PTR, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.qb_paged_attention(*a.values())


ARG, UNSUPPORTED = 1, 6
COMMON = [(dict(k=None), ARG), (dict(v=PTR + 2), ARG), (dict(table=None), ARG), (dict(q_start=None), ARG),
          (dict(kv=None), ARG), (dict(status=None), ARG), (dict(out=None), ARG), (dict(hq=12), ARG), (dict(hq=0), ARG),
          (dict(hkv=0), ARG), (dict(hq=136), UNSUPPORTED), (dict(hq=65, hkv=65), UNSUPPORTED),
          (dict(page=8), UNSUPPORTED), (dict(page=48), UNSUPPORTED), (dict(page=512), UNSUPPORTED),
          (dict(pages=0), UNSUPPORTED), (dict(pages=1 << 26), UNSUPPORTED), (dict(seqs=0), UNSUPPORTED),
          (dict(seqs=1025), UNSUPPORTED), (dict(width=0), UNSUPPORTED), (dict(width=1 << 27), UNSUPPORTED),
          (dict(tokens=-1), UNSUPPORTED)]


@pytest.mark.parametrize("kw,code", COMMON + [(dict(qkv=None), ARG), (dict(cos=None), ARG), (dict(sin=PTR + 8), ARG),
                                              (dict(rows=0), ARG), (dict(first=-1), ARG), (dict(qn=PTR + 4), ARG)])
def test_append_refuses(built_lib, kw, code):
    assert _append(built_lib, **kw) == code
    assert built_lib.qb_last_error(None)


@pytest.mark.parametrize("kw,code", COMMON + [(dict(q=None), ARG), (dict(window=-1), ARG), (dict(sinks=-1), ARG),
                                              (dict(max_q=-1), ARG), (dict(max_q=0), ARG), (dict(ws=None), ARG), (dict(ws_bytes=100), ARG), (dict(out=PTR + 16), ARG),
                                              (dict(ws=PTR + 128), ARG)])
def test_attention_refuses(built_lib, kw, code):
    assert _attention(built_lib, **kw) == code
    assert built_lib.qb_last_error(None)


def _prefix(lib, **kw):
    a = dict(q=PTR, k=PTR, v=PTR, pages=4, page=16, ptable=PTR, ppages=2, plen=20, table=PTR, width=4, q_start=PTR,
             kv=PTR, seqs=1, tokens=1, max_q=1, hq=16, hkv=8, out=PTR, ws=PTR, ws_bytes=1 << 40, status=PTR, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.qb_shared_prefix_attention(*a.values())


@pytest.mark.parametrize("kw,code", COMMON + [(dict(q=None), ARG), (dict(plen=-1), ARG), (dict(plen=33), ARG),
                                              (dict(ptable=None), ARG), (dict(ppages=-1), ARG), (dict(max_q=0), ARG),
                                              (dict(ws=None), ARG), (dict(ws_bytes=100), ARG)])
def test_shared_prefix_refuses(built_lib, kw, code):
    assert _prefix(built_lib, **kw) == code
    assert built_lib.qb_last_error(None)


def test_sizes_beyond_the_tile_counts_are_refused(built_lib):
    assert _attention(built_lib, tokens=1 << 24, max_q=1 << 24, hq=128) == UNSUPPORTED  # too many blocks of rows
    assert _attention(built_lib, seqs=1024, width=1 << 26) == UNSUPPORTED  # too many key tiles


def test_tensors_that_require_a_gradient_are_refused():
    from hackthenorth_b200 import ops

    q = torch.zeros(1, 16, 128, dtype=torch.bfloat16, requires_grad=True)
    for call in (lambda: ops.paged_attention(q, q, q, q, q, q), lambda: ops.shared_prefix_attention(q, q, q, q, 0, q, q, q),
                 lambda: ops.rope_paged_append(q, q, q, q, q, q, q, q, q, q), lambda: ops.sample_token(q, q)):
        with pytest.raises(ValueError, match="backward"):
            call()


def test_empty_calls_return_without_a_launch(built_lib):
    assert _append(built_lib, tokens=0, qkv=None, out=None) == 0
    assert _attention(built_lib, tokens=0, q=None, out=None) == 0
    assert _attention(built_lib, tokens=0, max_q=0) == 0
    assert _prefix(built_lib, tokens=0, q=None) == 0


def test_python_calls_refuse_cpu_tensors():
    from hackthenorth_b200 import ops

    z = torch.zeros(4, 8, 16, 128, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.paged_attention(torch.zeros(1, 16, 128, dtype=torch.bfloat16), z, z, i[None], i, i[:1])
    with pytest.raises(ValueError):
        ops.rope_paged_append(torch.zeros(1, 4096, dtype=torch.bfloat16), None, None, z[0, 0], z[0, 0], z, z, i[None], i,
                              i[:1])


@pytest.mark.parametrize("kw,code", [(dict(logits=None), ARG), (dict(logits=PTR + 1), ARG), (dict(fp32=1, logits=PTR + 2), ARG),
                                     (dict(uniforms=None), ARG), (dict(out=None), ARG), (dict(status=None), ARG),
                                     (dict(rows=-1), UNSUPPORTED), (dict(vocab=0), UNSUPPORTED),
                                     (dict(vocab=262145), UNSUPPORTED)])
def test_sample_refuses(built_lib, kw, code):
    a = dict(logits=PTR, fp32=0, rows=1, vocab=100, uniforms=PTR, t=None, t_all=1.0, k=None, k_all=0, p=None, p_all=1.0,
             m=None, m_all=0.0, out=PTR, status=PTR, stream=None)
    a.update(kw)
    assert built_lib.qb_sample_token(*a.values()) == code
    assert built_lib.qb_last_error(None)
    a.update(logits=None, rows=0, vocab=100)
    assert built_lib.qb_sample_token(*a.values()) == 0
