"""The paged key/value cache's entry points on the host (no GPU): descriptor
layouts against the header, refusals before any launch."""
import ctypes
import os
import re

import pytest
import torch

from fluxvla_amd import _lib
from fluxvla_amd import kernels as K

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                      'include', 'fluxvla_amd.h')


@pytest.mark.parametrize('name,mirror', [('fvx_paged_append_desc', _lib.PagedAppendDesc),
                                         ('fvx_paged_attn_desc', _lib.PagedAttnDesc)])
def test_desc_layout_matches_c(name, mirror):
    text = open(HEADER).read()
    body = text[text.index('typedef struct ' + name):]
    body = re.sub(r'/\*.*?\*/', '', body[:body.index('} ' + name + ';')], flags=re.S)
    assert re.findall(r'\*?\s*(\w+)\s*[;,]', body) == [f[0] for f in mirror._fields_]
    kinds = {'int64_t': ctypes.c_int64, 'int32_t': ctypes.c_int32, 'float': ctypes.c_float}
    fields = dict(mirror._fields_)
    for decl in re.findall(r'([^;{]+);', body.split('{', 1)[1]):
        kind = decl.replace('const', '').split()[0]
        for part in decl.split(','):
            nm = re.findall(r'\w+', part)[-1]
            want = ctypes.c_void_p if '*' in part else kinds[kind]
            assert fields[nm] is want, nm


def _append(**kw):
    d = _lib.PagedAppendDesc()
    d.qkv, d.ld_qkv, d.q_out, d.ld_q = 4096, 2560, 8192, 2048
    d.k, d.v, d.rope, d.max_pos = 16384, 32768, 65536, 100
    d.page_table, d.table_stride, d.kv_len = 4096, 4, 4096
    d.n_rows, d.n_seqs, d.max_pages = 2, 2, 4
    d.n_pages, d.page_size, d.q_heads, d.kv_heads, d.head_dim = 8, 16, 8, 1, 256
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _attn(**kw):
    d = _lib.PagedAttnDesc()
    d.q, d.ldq, d.o, d.ldo = 4096, 2048, 8192, 2048
    d.k, d.v = 16384, 32768
    d.page_table, d.table_stride, d.kv_len = 4096, 4, 4096
    d.n_rows, d.n_seqs, d.max_pages, d.max_q = 2, 2, 4, 1
    d.n_pages, d.page_size, d.q_heads, d.kv_heads, d.head_dim = 8, 16, 8, 1, 256
    d.scale = 0.0625
    for k, v in kw.items():
        setattr(d, k, v)
    return d


BOTH = [
    ({'head_dim': 72}, _lib.FVX_ERR_SHAPE, 'head_dim'),
    ({'page_size': 8}, _lib.FVX_ERR_SHAPE, 'page_size'),
    ({'page_size': 48}, _lib.FVX_ERR_SHAPE, 'page_size'),
    ({'page_size': 2048}, _lib.FVX_ERR_SHAPE, 'page_size'),
    ({'kv_heads': 0}, _lib.FVX_ERR_SHAPE, 'kv_heads'),
    ({'n_rows': -1}, _lib.FVX_ERR_SHAPE, 'negative'),
    ({'n_pages': 0}, _lib.FVX_ERR_SHAPE, 'n_pages'),
    ({'max_pages': 1 << 26}, _lib.FVX_ERR_SHAPE, '2^30'),
    ({'max_pages': 1 << 62}, _lib.FVX_ERR_SHAPE, '2^30'),
    ({'n_rows': 1 << 30, 'n_seqs': 1 << 30}, _lib.FVX_ERR_SHAPE, '2^30'),
    ({'n_rows': 3}, _lib.FVX_ERR_SHAPE, 'q_start'),
    ({'e4m3': 2}, _lib.FVX_ERR_ARG, 'e4m3'),
    ({'e4m3': 1}, _lib.FVX_ERR_NULL, 'k_scale'),
    ({'k': 0}, _lib.FVX_ERR_NULL, 'required'),
    ({'kv_len': 0}, _lib.FVX_ERR_NULL, 'required'),
    ({'page_table': 0}, _lib.FVX_ERR_NULL, 'required'),
    ({'v': 32776}, _lib.FVX_ERR_ALIGN, '16B'),
    ({'table_stride': 3}, _lib.FVX_ERR_SHAPE, 'table_stride'),
]


@pytest.mark.parametrize('kw,status,text', BOTH + [
    ({'q_heads': -1}, _lib.FVX_ERR_SHAPE, 'q_heads'),
    ({'rope': 0}, _lib.FVX_ERR_NULL, 'rope'),
    ({'ld_qkv': 2556}, _lib.FVX_ERR_ALIGN, 'multiples of 8'),
    ({'ld_qkv': 2552}, _lib.FVX_ERR_SHAPE, 'ld_qkv'),
    ({'ld_q': 2040}, _lib.FVX_ERR_SHAPE, 'ld_q'),
    ({'max_pos': -1}, _lib.FVX_ERR_SHAPE, 'max_pos'),
    ({'n_rows': 1 << 26, 'n_seqs': 1 << 26}, _lib.FVX_ERR_SHAPE, '2^26'),
])
def test_append_refuses(kw, status, text):
    lib = _lib.load()
    assert lib.fvx_paged_append(ctypes.byref(_append(**kw)), None) == status
    assert text in lib.fvx_last_error().decode()


@pytest.mark.parametrize('kw,status,text', BOTH + [
    ({'q_heads': 7, 'kv_heads': 2}, _lib.FVX_ERR_SHAPE, 'multiple'),
    ({'q_heads': 0}, _lib.FVX_ERR_SHAPE, 'q_heads'),
    ({'max_q': -1}, _lib.FVX_ERR_SHAPE, 'max_q'),
    ({'window': -1}, _lib.FVX_ERR_SHAPE, 'window'),
    ({'softcap': -1.0}, _lib.FVX_ERR_ARG, 'softcap'),
    ({'softcap': float('inf')}, _lib.FVX_ERR_ARG, 'softcap'),
    ({'scale': float('nan')}, _lib.FVX_ERR_ARG, 'scale'),
    ({'softcap': 1e-39}, _lib.FVX_ERR_ARG, 'too small'),
    ({'softcap': 1025.0}, _lib.FVX_ERR_ARG, '1024'),
    ({'ldq': 2044}, _lib.FVX_ERR_ALIGN, 'multiples of 8'),
    ({'ldo': 2040}, _lib.FVX_ERR_SHAPE, 'ldo'),
    ({}, _lib.FVX_ERR_WORKSPACE, 'workspace'),
    ({'workspace': 4096, 'workspace_bytes': 64}, _lib.FVX_ERR_WORKSPACE, 'workspace'),
])
def test_attention_refuses(kw, status, text):
    lib = _lib.load()
    assert lib.fvx_paged_attention(ctypes.byref(_attn(**kw)), None) == status
    assert text in lib.fvx_last_error().decode()


def test_null_descriptors_and_empty_batches():
    lib = _lib.load()
    assert lib.fvx_paged_append(None, None) == _lib.FVX_ERR_NULL
    assert lib.fvx_paged_attention(None, None) == _lib.FVX_ERR_NULL
    assert lib.fvx_paged_attention_workspace_bytes(None) == _lib.FVX_ERR_NULL
    assert lib.fvx_paged_attention_workspace_bytes(
        ctypes.byref(_attn(head_dim=72))) == _lib.FVX_ERR_SHAPE
    assert lib.fvx_paged_attention_workspace_bytes(ctypes.byref(_attn())) > 0
    empty = {'n_rows': 0, 'n_seqs': 0}
    assert lib.fvx_paged_append(ctypes.byref(_append(**empty)), None) == 0
    assert lib.fvx_paged_attention(ctypes.byref(_attn(**empty)), None) == 0
    assert lib.fvx_paged_attention_workspace_bytes(ctypes.byref(_attn(**empty))) == 0


def test_head_rows():
    t = torch.zeros(6, 8, 64)
    assert K._head_rows(t, 't', 8, 64) == (6, 512)
    assert K._head_rows(t.view(6, 512), 't', 8, 64) == (6, 512)
    assert K._head_rows(torch.zeros(6, 1024)[:, :512], 't', 8, 64) == (6, 1024)
    assert K._head_rows(t[:1], 't', 8, 64) == (1, 512)
    for bad in (t.transpose(0, 1), t[..., ::2], torch.zeros(6, 4, 64),
                torch.zeros(1, 512).expand(6, 512), torch.zeros(6, 8, 128)[..., :64]):
        with pytest.raises(ValueError):
            K._head_rows(bad, 't', 8, 64)


def test_host_tensors_are_refused():
    k, v = torch.zeros(2, 1, 16, 64).bfloat16(), torch.zeros(2, 1, 64, 16).bfloat16()
    with pytest.raises(ValueError, match='CUDA'):
        K.PagedKV(k, v)
