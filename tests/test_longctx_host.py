"""The long-context operators' boundary without a GPU: the binding's structures lie as the header's, and calls
without a context or a descriptor are refused."""
import ctypes as C
import os
import subprocess

import pytest

import ork_b200 as B

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PAIRS = [("ork_b200_attn", B.Attn), ("ork_b200_kv4", B.KV4), ("ork_b200_kv4_attn", B.KV4Attn), ("ork_b200_evict", B.Evict)]


def test_structures_lie_as_the_headers(tmp_path):
    src = '#include <stdio.h>\n#include <stddef.h>\n#define ORK_F16_AS_U16\n#include "ork_b200.h"\nint main(void) {\n'
    for name, st in PAIRS:
        src += f'printf("%zu", sizeof({name}));\n'
        src += "".join(f'printf(" %zu", offsetof({name}, {f[0]}));\n' for f in st._fields_) + 'printf("\\n");\n'
    (tmp_path / "a.c").write_text(src + "return 0; }\n")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(tmp_path / "a"), str(tmp_path / "a.c")], check=True)
    got = subprocess.run([str(tmp_path / "a")], capture_output=True, text=True, check=True).stdout.split("\n")
    for (name, st), line in zip(PAIRS, got):
        assert [int(x) for x in line.split()] == [C.sizeof(st)] + [getattr(st, f[0]).offset for f in st._fields_], name


@pytest.mark.parametrize("name,args", [
    ("ork_b200_attn_async", (None, C.byref(B.Attn()))),
    ("ork_b200_kv4_attn_async", (None, C.byref(B.KV4()), C.byref(B.KV4Attn()))),
    ("ork_b200_kv4_store_async", (None, C.byref(B.KV4()), None, None, 0, 1, 64, 64, None, None)),
    ("ork_b200_kv4_load_async", (None, C.byref(B.KV4()), None, None, 0, 1, 64, 64, None, None)),
    ("ork_b200_evict_async", (None, C.byref(B.Evict())))])
def test_no_context_is_refused(name, args):
    assert getattr(B.lib(), name)(*args) == -1


def test_types_are_the_headers():
    src = open(os.path.join(ROOT, "include", "ork_b200.h")).read()
    for n, v in B.TYPES.items():
        assert f"#define ORK_B200_{n.upper()} {v}\n" in src
    assert f"#define ORK_B200_EVICT_PLANES {len(B.Evict().src)}\n" in src
