"""The forward operators' header and binding, without a GPU: the header is plain C, every function it declares is bound
with as many arguments as it has, and null handles are refused with a message."""
import ctypes
import importlib
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def declarations():
    src = open(os.path.join(ROOT, "include", "dpb_forward.h")).read()
    src = re.sub(r"/\*.*?\*/", "", src, flags=re.S)
    return {m.group(1): [a for a in m.group(2).split(",")] for m in re.finditer(r"\b(dpb_[a-z0-9_]+)\s*\(([^)]*)\)\s*;", src)}


def test_header_is_c(tmp_path):
    f = tmp_path / "t.c"
    f.write_text('#include "dpb_forward.h"\nint main(void) { return 0; }\n')
    r = subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-pedantic", "-fsyntax-only", "-I", os.path.join(ROOT, "include"), str(f)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


def test_binding_covers_the_header(dpb):
    fw = importlib.import_module("deep_prove_b200.forward")
    decl = declarations()
    assert set(decl) == set(fw.FORWARD_SIGNATURES)
    for name, args in decl.items():
        assert len(args) == len(fw.FORWARD_SIGNATURES[name][1]), name


@pytest.mark.parametrize("name", ["dpb_embedding_lookup", "dpb_row_groups_new", "dpb_row_groups_sum", "dpb_expert_weights_new",
                                  "dpb_grouped_product"])
def test_null_handles_are_refused(dpb, name):
    fw = importlib.import_module("deep_prove_b200.forward")
    out = ctypes.c_void_p()
    args = [None if t is ctypes.c_void_p else ctypes.byref(out) if t is fw._pp else 1 for t in fw.FORWARD_SIGNATURES[name][1]]
    assert getattr(dpb.lib, name)(*args) == dpb.EINVAL
    assert b"null argument" in dpb.lib.dpb_last_error() and not out.value


def test_null_handles_are_freed_quietly(dpb):
    importlib.import_module("deep_prove_b200.forward")
    dpb.lib.dpb_row_groups_free(None)
    dpb.lib.dpb_expert_weights_free(None)
    assert dpb.lib.dpb_row_groups_len(None) == 0
