"""CPU checks of attention and the key-value cache: arguments are refused
before any device work (status 1 with a message), sizes of workspaces, struct
layouts, and no CPU fallback in the Python functions."""

from __future__ import annotations

import ctypes
import subprocess

import pytest

from conftest import ROOT, pkg, submodule

FAKE = 1 << 20  # never dereferenced: every call here is refused or has nothing to do


@pytest.fixture(scope="module")
def N():
    return submodule("_native")


@pytest.fixture(scope="module")
def libso(N):
    return N.load_library()


def _rows(N, data=FAKE, token=512, head=64):
    return N.HeadRows(data, token, head)


def _attention(N, **changes):
    d = N.Attention(tokens=32, keys=32, sequences=2, heads=8, kv_heads=2, head_dim=64, q=_rows(N), k=_rows(N), v=_rows(N),
                    offsets=FAKE, key_offsets=FAKE, out=FAKE, lse=FAKE, d_out=_rows(N), d_q=FAKE, d_k=FAKE, d_v=FAKE,
                    workspace=FAKE, workspace_bytes=1 << 30, causal=1, scale=0.125)
    for name, value in changes.items():
        setattr(d, name, value)
    return ctypes.byref(d)


SHAPES = [
    (dict(tokens=-1), "invalid shape"), (dict(keys=-1), "invalid shape"), (dict(heads=7), "multiple"),
    (dict(kv_heads=0), "multiple"), (dict(heads=0), "multiple"), (dict(heads=131072), "65536"),
    (dict(head_dim=0), "head_dim"), (dict(head_dim=60), "head_dim"), (dict(head_dim=264), "head_dim"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(tokens=1 << 28), "2^30"), (dict(keys=1 << 28), "2^30"),
    (dict(sequences=0), "sequences"), (dict(sequences=1 << 24), "sequences"), (dict(offsets=None), "key_offsets"),
    (dict(offsets=None, key_offsets=None, keys=33), "key_offsets"),
    (dict(offsets=FAKE, key_offsets=None, keys=33), "key_offsets"),
    (dict(sequences=(1 << 23)), "grid"), (dict(out=None), "null"), (dict(out=FAKE + 8), "aligned"),
]


@pytest.mark.parametrize("changes, message", SHAPES)
def test_attention_refusals(N, libso, changes, message):
    for call in (libso.glm53_packed_attention, libso.glm53_packed_attention_backward):
        assert call(_attention(N, **changes), None) == N.INVALID_ARGUMENT
        assert message in libso.glm53_last_error().decode()


@pytest.mark.parametrize("rows, message", [
    ((None, 512, 64), "null"), ((FAKE + 2, 512, 64), "aligned"), ((FAKE, 508, 64), "stride"), ((FAKE, 512, 60), "stride"),
    ((FAKE, -512, 64), "stride"), ((FAKE, 1 << 23, 64), "stride"), ((FAKE, 512, 1 << 23), "stride"),
])
def test_row_refusals(N, libso, rows, message):
    for name in ("q", "k", "v"):
        assert libso.glm53_packed_attention(_attention(N, **{name: N.HeadRows(*rows)}), None) == N.INVALID_ARGUMENT
        assert message in libso.glm53_last_error().decode() and name in libso.glm53_last_error().decode()
    assert libso.glm53_packed_attention_backward(_attention(N, d_out=N.HeadRows(*rows)), None) == N.INVALID_ARGUMENT
    assert message in libso.glm53_last_error().decode()


@pytest.mark.parametrize("changes, message", [
    (dict(lse=None), "lse"), (dict(d_q=FAKE + 8), "aligned"), (dict(d_v=FAKE + 4), "aligned"),
    (dict(workspace=None), "workspace"), (dict(workspace=FAKE + 16), "workspace"), (dict(workspace_bytes=2047), "workspace"),
])
def test_attention_backward_refusals(N, libso, changes, message):
    assert libso.glm53_packed_attention_backward(_attention(N, **changes), None) == N.INVALID_ARGUMENT
    assert message in libso.glm53_last_error().decode()


def test_attention_without_rows_and_workspace_sizes(N, libso):
    assert libso.glm53_packed_attention(None, None) == N.INVALID_ARGUMENT
    assert libso.glm53_packed_attention_backward(None, None) == N.INVALID_ARGUMENT
    assert libso.glm53_packed_attention(_attention(N, tokens=0, out=None, q=N.HeadRows(None, 0, 0)), None) == N.OK
    size = libso.glm53_packed_attention_backward_workspace_bytes
    assert size(0, 8) == size(8, 0) == size(1 << 28, 8) == 0
    assert size(32, 8) == 2048 and size(33, 8) == 2304
    paged = libso.glm53_paged_attention_workspace_bytes
    assert paged(0, 0) == paged(257, 0) == 0
    assert 0 < paged(64, 0) <= paged(128, 1) <= paged(256, 1) < 1 << 26


def test_split_bytes(libso):
    """Parts of few key heads' gradients: FP32 [splits, keys, kv_heads, dim] of d_k and d_v."""
    size = libso.glm53_packed_attention_backward_split_bytes
    for refused in ((0, 8, 1, 8, 1, 64), (8, 0, 1, 8, 1, 64), (1 << 28, 8, 1, 8, 1, 64), (4096, 4096, 1, 8, 3, 64),
                    (4096, 4096, 1, 8, 0, 64), (4096, 4096, 1, 8, 1, 512), (4096, 4096, 1 << 24, 8, 1, 64)):
        assert size(*refused) == 0
    assert size(8192, 8192, 1, 8, 1, 128) == 8 * 8192 * 128 * 8  # 128 tiles
    assert size(8192, 8192, 0, 8, 1, 128) == size(8192, 8192, 1, 8, 1, 128)  # no offsets
    assert size(8192, 8192, 30, 8, 1, 128) == 0  # short sequences
    assert size(4096, 4096, 1, 16, 8, 128) == 0  # tiles enough
    assert size(100, 100, 1, 8, 1, 128) == 0


def _cache(N, **changes):
    c = N.KVCache(k_pages=FAKE, v_pages=FAKE, k_scales=None, v_scales=None, page_table=FAKE, pages=4, page_size=16, kv_heads=2,
                  head_dim=64, sequences=3, max_pages=2, table_stride=2, e4m3=0)
    for name, value in changes.items():
        setattr(c, name, value)
    return c


CACHES = [
    (dict(kv_heads=0), "heads"), (dict(head_dim=4), "head_dim"), (dict(head_dim=512), "head_dim"), (dict(pages=0), "pages"),
    (dict(pages=1 << 31), "pages"), (dict(page_size=8), "page_size"), (dict(page_size=48), "page_size"),
    (dict(page_size=1 << 17), "page_size"), (dict(sequences=-1), "sequences"), (dict(sequences=1 << 24), "sequences"),
    (dict(max_pages=-1), "page table"), (dict(table_stride=1), "page table"), (dict(k_pages=None), "null"),
    (dict(v_pages=None), "null"), (dict(page_table=None), "null"), (dict(v_pages=FAKE + 8), "aligned"),
    (dict(k_scales=FAKE), "scales"), (dict(e4m3=1), "scales"), (dict(e4m3=1, k_scales=FAKE, v_scales=FAKE + 4), "aligned"),
    (dict(e4m3=1, k_scales=FAKE, v_scales=FAKE, head_dim=72), "multiple of 16"),
]


def _append(N, libso, cache, k=None, tokens=3, offsets=None, lengths=FAKE):
    k = _rows(N) if k is None else k
    return libso.glm53_kv_append(ctypes.byref(cache), ctypes.byref(k), ctypes.byref(_rows(N)), tokens, offsets, lengths, None)


def _paged(N, libso, cache, q=None, heads=4, lengths=FAKE, scale=0.125, out=FAKE, ws=FAKE, ws_bytes=1 << 30):
    q = _rows(N) if q is None else q
    return libso.glm53_paged_attention(ctypes.byref(cache), ctypes.byref(q), heads, lengths, scale, out, ws, ws_bytes, None)


@pytest.mark.parametrize("changes, message", CACHES)
def test_cache_refusals(N, libso, changes, message):
    cache = _cache(N, **changes)
    for call in (lambda: _append(N, libso, cache), lambda: _paged(N, libso, cache),
                 lambda: libso.glm53_kv_read(ctypes.byref(cache), FAKE, 8, FAKE, FAKE, None)):
        assert call() == N.INVALID_ARGUMENT
        assert message in libso.glm53_last_error().decode()


def test_append_read_and_paged_refusals(N, libso):
    cache = _cache(N)

    def refused(status, message):
        assert status == N.INVALID_ARGUMENT
        assert message in libso.glm53_last_error().decode(), libso.glm53_last_error()

    refused(_append(N, libso, cache, tokens=-1), "tokens")
    refused(_append(N, libso, cache, tokens=4), "one token a sequence")
    refused(_append(N, libso, cache, lengths=None), "lengths")
    refused(_append(N, libso, cache, k=N.HeadRows(FAKE + 2, 128, 64)), "aligned")
    refused(libso.glm53_kv_append(ctypes.byref(cache), None, ctypes.byref(_rows(N)), 3, None, FAKE, None), "null")
    refused(libso.glm53_kv_read(ctypes.byref(cache), None, 8, FAKE, FAKE, None), "offsets")
    refused(libso.glm53_kv_read(ctypes.byref(cache), FAKE, -1, FAKE, FAKE, None), "rows")
    refused(libso.glm53_kv_read(ctypes.byref(cache), FAKE, 8, FAKE + 4, FAKE, None), "aligned")
    refused(libso.glm53_kv_read(None, FAKE, 8, FAKE, FAKE, None), "null")
    refused(_paged(N, libso, cache, heads=3), "multiple")
    refused(_paged(N, libso, cache, scale=0.0), "scale")
    refused(_paged(N, libso, cache, lengths=None), "null")
    refused(_paged(N, libso, cache, out=FAKE + 8), "aligned")
    refused(_paged(N, libso, cache, ws=None), "workspace")
    refused(_paged(N, libso, cache, ws_bytes=1024), "workspace")
    refused(_paged(N, libso, cache, ws=FAKE + 64), "workspace")
    refused(_paged(N, libso, _cache(N, sequences=1 << 22)), "sequences times heads")
    # nothing to do
    empty = _cache(N, sequences=0, page_table=None)
    assert _append(N, libso, empty, tokens=0) == N.OK
    assert _paged(N, libso, empty) == N.OK
    assert libso.glm53_kv_read(ctypes.byref(cache), None, 0, FAKE, FAKE, None) == N.OK


def test_limits_of_offsets_and_grids(N, libso):
    """What 32-bit offsets, a grid and the gradients' start values hold."""
    far = N.HeadRows(FAKE, 512, 1 << 22)
    for call in (libso.glm53_packed_attention, libso.glm53_packed_attention_backward):
        assert call(_attention(N, heads=512, kv_heads=512, q=far), None) == N.INVALID_ARGUMENT
        assert "apart" in libso.glm53_last_error().decode()
        assert call(_attention(N, scale=2.0**-65), None) == N.INVALID_ARGUMENT
        assert "scale" in libso.glm53_last_error().decode()
    assert _paged(N, libso, _cache(N), heads=512, q=far) == N.INVALID_ARGUMENT
    assert "apart" in libso.glm53_last_error().decode()
    cache = _cache(N)
    assert _append(N, libso, cache, tokens=1 << 25, offsets=FAKE) == N.INVALID_ARGUMENT
    assert "tokens" in libso.glm53_last_error().decode()
    assert libso.glm53_kv_read(ctypes.byref(cache), FAKE, 1 << 25, FAKE, FAKE, None) == N.INVALID_ARGUMENT
    assert "rows" in libso.glm53_last_error().decode()


def test_struct_layouts(N, tmp_path):
    structs = {"glm53_head_rows": N.HeadRows, "glm53_attention": N.Attention, "glm53_kv_cache": N.KVCache}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{ROOT / "include" / "glm53_moe.h"}"', "int main(void) {"]
    for name, kind in structs.items():
        lines.append(f'  printf("{name} sizeof %zu\\n", sizeof({name}));')
        lines += [f'  printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in kind._fields_]
    (tmp_path / "layout.c").write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", "-o", str(tmp_path / "layout"), str(tmp_path / "layout.c")], check=True)
    for line in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.splitlines():
        name, field, value = line.split()
        kind = structs[name]
        assert int(value) == (ctypes.sizeof(kind) if field == "sizeof" else getattr(kind, field).offset), line


def test_no_cpu_fallback():
    import torch

    M = pkg()
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    pages = torch.zeros(2, 2, 16, 64, dtype=torch.bfloat16)
    table, lengths = torch.zeros(4, 1, dtype=torch.int32), torch.ones(4, dtype=torch.int32)
    for call in (lambda: M.packed_attention(q, q, q), lambda: M.paged_attention(q, pages, pages, table, lengths),
                 lambda: M.append_kv(q, q, pages, pages, table, lengths),
                 lambda: M.read_kv(pages, pages, table, torch.arange(5, dtype=torch.int32), 4)):
        with pytest.raises((RuntimeError, ValueError), match="ROCm"):
            call()


def test_batch_refusals():
    import torch

    M = pkg()
    i = torch.zeros(3, dtype=torch.int32)
    table = torch.zeros(2, 1, dtype=torch.int32)
    for wrong in (dict(), dict(page_table=table), dict(lengths=i), dict(offsets=i, key_offsets=i, keys=3),
                  dict(offsets=i, page_table=table, lengths=i, key_offsets=i),
                  dict(page_table=table, lengths=i, key_offsets=i, keys=3)):
        with pytest.raises(ValueError):
            M.AttentionBatch(**wrong)
    assert torch.equal(M.AttentionBatch(page_table=table, lengths=i).after, i + 1)
    with pytest.raises(ValueError, match="multiple"):
        M.SelfAttention(64, 4, 3)
