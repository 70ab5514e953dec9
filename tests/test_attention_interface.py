"""The attention and cache interface without a GPU: descriptor layouts, and the Python form's checks of arguments."""

import ctypes
import os
import subprocess

import pytest

torch = pytest.importorskip("torch")

from tosa_b200 import _lib as L  # noqa: E402
from tosa_b200.attention import PagedCache, attention  # noqa: E402

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "tosa_b200.h")


def test_descriptor_layouts(tmp_path):
    structs = {"tb_attention_desc": L.AttentionDesc, "tb_cache_desc": L.CacheDesc, "tb_cache_buffers": L.CacheBuffers}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {"]
    for name, py in structs.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in py._fields_]
    lines.append('printf("pages %d\\n", TB_ERR_OUT_OF_PAGES); return 0; }')
    (tmp_path / "layout.c").write_text("\n".join(lines))
    subprocess.check_call(["gcc", "-std=c99", "-o", str(tmp_path / "layout"), str(tmp_path / "layout.c")])
    got = dict(x.split() for x in subprocess.check_output([str(tmp_path / "layout")]).decode().splitlines())
    for name, py in structs.items():
        assert int(got[name]) == ctypes.sizeof(py)
        for f, _ in py._fields_:
            assert int(got[f"{name}.{f}"]) == getattr(py, f).offset, f
    assert int(got["pages"]) == L.TB_ERR_OUT_OF_PAGES and L.STATUS_NAMES[L.TB_ERR_OUT_OF_PAGES] == "OutOfPages"


def _qkv(**kw):
    t = dict(q=torch.zeros(4, 2, 64).half(), k=torch.zeros(6, 1, 64).half(), v=torch.zeros(6, 1, 64).half(),
             cu_q=torch.tensor([0, 4], dtype=torch.int32), cu_k=torch.tensor([0, 6], dtype=torch.int32))
    t.update(kw)
    return t


@pytest.mark.parametrize("change,kind", [
    (dict(q=torch.zeros(4, 2, 64)), "DTypeMismatch"),
    (dict(k=torch.zeros(6, 1, 64).bfloat16()), "DTypeMismatch"),
    (dict(k=torch.zeros(6, 1, 32).half()), "ShapeMismatch"),
    (dict(v=torch.zeros(5, 1, 64).half()), "ShapeMismatch"),
    (dict(v=torch.zeros(6, 2, 64).half()), "ShapeMismatch"),
    (dict(q=torch.zeros(4, 128).half()), "ShapeMismatch"),
    (dict(q=torch.zeros(4, 64, 2).half().transpose(1, 2)), "ShapeMismatch"),
    (dict(cu_q=torch.tensor([0, 4])), "ShapeMismatch"),
    (dict(cu_k=torch.tensor([0, 3, 6], dtype=torch.int32)), "ShapeMismatch"),
    (dict(cu_q=torch.zeros(0, dtype=torch.int32), cu_k=torch.zeros(0, dtype=torch.int32)), "ShapeMismatch"),
    (dict(out=torch.zeros(4, 2, 64)), "DTypeMismatch"),
    (dict(out=torch.zeros(4, 1, 64).half()), "ShapeMismatch"),
    (dict(lse=torch.zeros(4, 2)), "ShapeMismatch"),
])
def test_attention_refuses(change, kind):
    with pytest.raises(L.TbError) as e:
        attention(None, **_qkv(**change))
    assert e.value.kind == kind


@pytest.mark.parametrize("change,kind", [
    (dict(k_pages=torch.zeros(1, 4, 1, 8, 64)), "DTypeMismatch"),
    (dict(v_pages=torch.zeros(1, 4, 1, 8, 64).bfloat16()), "DTypeMismatch"),
    (dict(v_pages=torch.zeros(1, 5, 1, 8, 64).half()), "ShapeMismatch"),
    (dict(lengths=torch.zeros(4, dtype=torch.int32)), "ShapeMismatch"),
    (dict(refs=torch.zeros(5, dtype=torch.int32)), "ShapeMismatch"),
    (dict(refs=torch.zeros(4)), "DTypeMismatch"),
    (dict(), "InvalidArgument"),  # not on a GPU
])
def test_cache_refuses(change, kind):
    t = dict(k_pages=torch.zeros(1, 4, 1, 8, 64).half(), v_pages=torch.zeros(1, 4, 1, 8, 64).half(),
             page_table=torch.zeros(3, 4, dtype=torch.int32), lengths=torch.zeros(3, dtype=torch.int32),
             refs=torch.zeros(4, dtype=torch.int32))
    t.update(change)
    with pytest.raises(L.TbError) as e:
        PagedCache(None, **t)
    assert e.value.kind == kind
