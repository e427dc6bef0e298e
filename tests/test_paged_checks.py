"""CPU: what the calls over the paged cache refuse, before anything runs on a device; layout of their descriptors."""
import ctypes
import os
import subprocess

import pytest

from mm_amx_b200 import capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 0x10000          # an aligned address that nothing reads


def cache(**kw):
    c = dict(pages=4, page_tokens=16, Hkv=2, D=64, dtype=capi.BF16, k=A, v=A, page_stride=4096, head_stride=2048, token_stride=128, k_scale=None, v_scale=None,
             scale_page_stride=0, B=2, max_pages=2, page_table=A, table_stride=8, seq_lens=A)
    c.update(kw)
    return capi.PagedCache(**c)


def s8(**kw):
    return cache(**dict(dict(dtype=capi.S8, k_scale=A, v_scale=A, scale_page_stride=8), **kw))


def append(c, **kw):
    a = dict(cache=capi.pointer(c), T=2, k=A, k_row_stride=256, k_head_stride=128, v=A, v_row_stride=256, v_head_stride=128, H=4, q=A, q_row_stride=512,
             q_head_stride=128, q_out=A, q_out_row_stride=512, q_out_head_stride=128, rot_dim=64, rot_positions=10, rot_cos=A, rot_sin=A, rot_stride=128, axes=1)
    a.update(kw)
    return capi.kv_append(capi.KvAppend(**a))


def attend(c, **kw):
    a = dict(cache=capi.pointer(c), T=2, max_rows=1, H=4, q=A, q_row_stride=512, q_head_stride=128, out=2 * A, out_row_stride=512, out_head_stride=128, scale=1.0)
    a.update(kw)
    return capi.paged_attention(capi.PagedAttention(**a))


BAD_CACHE = [dict(D=96), dict(D=0), dict(page_tokens=0), dict(page_tokens=24), dict(page_tokens=256), dict(dtype=capi.F32), dict(dtype=capi.U8), dict(pages=-1), dict(B=-1),
             dict(max_pages=-1), dict(Hkv=0), dict(Hkv=70000), dict(k=None), dict(v=None), dict(page_table=None), dict(seq_lens=None), dict(k=A + 8), dict(v=A + 2),
             dict(page_stride=4100), dict(head_stride=8), dict(token_stride=136), dict(token_stride=112), dict(page_stride=-4096), dict(head_stride=-2048),
             dict(token_stride=-128), dict(table_stride=4), dict(table_stride=10), dict(page_table=A + 2), dict(seq_lens=A + 1), dict(B=1), dict(B=3), dict(B=1 << 21)]
BAD_S8 = [dict(k_scale=None), dict(v_scale=None), dict(k_scale=A + 2), dict(scale_page_stride=4), dict(scale_page_stride=10)]
BAD_APPEND = [dict(k=None), dict(v=None), dict(q_out=None), dict(H=0), dict(H=-1), dict(T=-1), dict(k=A + 8), dict(v=A + 2), dict(q=A + 4), dict(q_out=A + 8), dict(k_row_stride=40),
              dict(v_head_stride=130), dict(q_head_stride=8), dict(q_out_row_stride=520), dict(q_out_row_stride=1024), dict(rot_dim=-16), dict(rot_dim=24), dict(rot_dim=80),
              dict(rot_cos=None), dict(rot_sin=None), dict(rot_positions=0), dict(rot_cos=A + 4), dict(rot_sin=A + 8), dict(rot_stride=112), dict(rot_stride=136), dict(axes=0),
              dict(axes=2), dict(axes=4), dict(axes=3, section=(capi.c_int * 3)(10, 10, 10)), dict(axes=3, section=(capi.c_int * 3)(40, -8, 0)), dict(positions=A + 2),
              dict(axes=3, section=(capi.c_int * 3)(16, 8, 8), positions=A, position_stride=4), dict(row_start=A + 1)]
BAD_ATTEND = [dict(q=None), dict(out=None), dict(H=0), dict(H=3), dict(H=70000), dict(T=-1), dict(max_rows=-1), dict(max_rows=0), dict(q=A + 8), dict(out=A + 2), dict(q_row_stride=520),
              dict(out_head_stride=8), dict(window=-1), dict(sinks=-1), dict(row_start=A + 2), dict(T=1), dict(T=3), dict(out=A),
              dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=-float("inf")), dict(scale=3e38)]


def refused(call, *args, **kw):
    with pytest.raises(capi.B200FCError) as e:
        call(*args, **kw)
    assert e.value.code in (capi.ERR_INVALID, capi.ERR_UNSUPPORTED), str(e.value)
    return str(e.value)


@pytest.mark.parametrize("kw", BAD_CACHE, ids=str)
def test_caches(kw):
    assert "kv_append" in refused(append, cache(**kw))
    assert "paged_attention" in refused(attend, cache(**kw))


@pytest.mark.parametrize("kw", BAD_S8, ids=str)
def test_factors_of_an_8_bit_cache(kw):
    refused(append, s8(**kw))
    refused(attend, s8(**kw))


@pytest.mark.parametrize("kw", BAD_APPEND, ids=str)
def test_append(kw):
    refused(append, cache(), **kw)


@pytest.mark.parametrize("kw", BAD_ATTEND, ids=str)
def test_attention(kw):
    refused(attend, cache(), **kw)


def test_null_descriptors_and_caches():
    assert capi.lib().b200fc_kv_append(None, None) == capi.ERR_INVALID
    assert capi.lib().b200fc_paged_attention(None, None) == capi.ERR_INVALID
    refused(lambda: capi.kv_append(capi.KvAppend()))
    refused(lambda: capi.paged_attention(capi.PagedAttention()))


def test_nothing_to_do_needs_no_device():
    append(cache(B=0), T=0)
    attend(cache(B=0), T=0)
    append(cache(B=3), T=0, row_start=A)
    attend(cache(B=3), T=0, row_start=A)


def test_layouts_match_the_header(tmp_path):
    names = {"b200fc_paged_cache_t": capi.PagedCache, "b200fc_kv_append_t": capi.KvAppend, "b200fc_paged_attention_t": capi.PagedAttention}
    src = tmp_path / "layout.c"
    lines = ['printf("%%zu\\n", sizeof(%s));' % n for n in names]
    lines += ['printf("%%zu\\n", offsetof(%s, %s));' % (n, f) for n, t in names.items() for f, _ in t._fields_]
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "b200fc.h"\nint main(void) { %s return 0; }\n' % " ".join(lines))
    exe = str(tmp_path / "layout")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    got = [int(v) for v in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(t) for t in names.values()] + [getattr(t, f).offset for t in names.values() for f, _ in t._fields_]
