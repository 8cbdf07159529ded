"""The decoder layer's C ABI without a GPU: exports, struct layouts, null contexts."""
import ctypes as C
import subprocess

import c4s


def test_exports_every_layer_symbol():
    names = c4s.header_functions(c4s.LAYERS_HEADER)
    assert sorted(names) == ["c4s_attn", "c4s_block_norm", "c4s_kv_append", "c4s_kv_read", "c4s_linear"]
    for n in names:
        assert hasattr(c4s.lib(), n)


def test_null_context_is_einval():
    L = c4s.lib()
    for n in ("c4s_block_norm", "c4s_linear"):
        assert getattr(L, n)(None, None, None) == c4s.EINVAL
    for n in ("c4s_kv_append", "c4s_kv_read", "c4s_attn"):
        assert getattr(L, n)(None, None, None, None) == c4s.EINVAL


def test_ctypes_structs_match_the_header(tmp_path):
    structs = {"c4s_norm": c4s.Norm, "c4s_linear_desc": c4s.Linear, "c4s_kv_cache": c4s.KvCacheDesc,
               "c4s_kv_rows": c4s.KvRows, "c4s_attn_desc": c4s.Attn}
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{c4s.LAYERS_HEADER}"', "int main(void) {"]
    for cname, py in structs.items():
        lines.append(f'  printf("{cname} size %zu\\n", sizeof({cname}));')
        for fname, _ in py._fields_:
            lines.append(f'  printf("{cname} {fname} %zu\\n", offsetof({cname}, {fname}));')
    lines += ["  return 0;", "}"]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines) + "\n")
    subprocess.run(["gcc", "-std=c11", "-o", str(exe), str(src)], check=True)
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split("\n"):
        if line:
            cname, what, val = line.split()
            py = structs[cname]
            assert int(val) == (C.sizeof(py) if what == "size" else getattr(py, what).offset), line
