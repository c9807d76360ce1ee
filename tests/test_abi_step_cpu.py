"""CPU-side checks of the step's entry points: the Python structures have the headers' layout, and null handles are refused."""
import ctypes as C
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layouts(tmp_path):
    from kore_amd import layer, paged, rope
    pairs = [("kore_rope_heads", rope.HeadsStruct), ("kore_paged_plan", paged.PlanStruct), ("kore_paged_rows", paged.RowsStruct),
             ("kore_paged_tree", paged.TreeStruct), ("kore_paged_keep", paged.KeepStruct), ("kore_layer_paged_opts", layer._PagedOpts)]
    src, want = tmp_path / "t.c", []
    lines = []
    for name, cls in pairs:
        lines.append('printf("%%zu ", sizeof(%s));' % name)
        want.append(C.sizeof(cls))
        for f, _ in cls._fields_:
            lines.append('printf("%%zu ", offsetof(%s, %s));' % (name, f))
            want.append(getattr(cls, f).offset)
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "kore_layer.h"\nint main(void) { %s return 0; }\n' % " ".join(lines))
    exe = tmp_path / "t"
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), "-o", str(exe), str(src)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == want


def test_null_handles():
    from kore_amd import layer, paged, rope
    L, bad = paged.lib(), rope.KORE_PAGED_E_INVALID
    assert L.kore_rope_norm_dev(None, 0, 1, 8, None, None, None, 1e-6, None) == bad
    assert L.kore_paged_plan_dev(None, None, None) == bad and L.kore_paged_keep_dev(None, None, None) == bad
    assert L.kore_paged_append_rows_dev(None, 0, None, 0, None, 0, None, 0, None, 0, None, 0, None) == bad
    assert L.kore_paged_attend_tree_dev(None, 0, None, None, 0, None, 0, None, 0, 0.0, 0, None, None) == bad
    assert b"null handle" in L.kore_paged_last_error(None)
    assert layer.lib().kore_layer_paged_ex_dev(None, None, None, 0, None, None, None, None, None) == layer.KORE_LAYER_E_INVALID
