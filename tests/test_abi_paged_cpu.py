"""CPU-side checks of libkore_paged.so: it exports what its headers declare and nothing else, and refuses bad configurations
before it touches a GPU."""
import ctypes as C
import os
import re
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADERS = [os.path.join(ROOT, "include", h) for h in ("kore_paged.h", "kore_rope.h")]


def _declared():
    names = set()
    for h in HEADERS:
        text = re.sub(r"/\*.*?\*/", "", open(h).read(), flags=re.S)
        names |= set(re.findall(r"\b(kore_(?:paged|rope)_[a-z_]+)\s*\(", text))
    return names


def test_exports_are_the_headers():
    from kore_amd import paged, rope
    L = paged.lib()
    out = subprocess.run(["nm", "-D", "--defined-only", rope.LIB_PATH], capture_output=True, text=True, check=True).stdout
    exported = {line.split()[-1] for line in out.splitlines() if " T " in line}
    assert {f for f in exported if "kore" in f} == _declared()
    assert {n for n, _, _ in rope.SYMBOLS + paged.SYMBOLS} == _declared()
    assert all(getattr(L, n) for n in _declared())


def test_headers_are_plain_c(tmp_path):
    src = tmp_path / "t.c"
    src.write_text('#include "kore_paged.h"\n#include "kore_attn.h"\nint main(void) { kore_paged_config c = {0}; return c.n_layer; }\n')
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), "-fsyntax-only", str(src)], check=True)


def test_struct_sizes(tmp_path):
    """The Python structures have the headers' sizes."""
    from kore_amd import paged, rope
    src = tmp_path / "t.c"
    src.write_text('#include <stdio.h>\n#include "kore_paged.h"\nint main(void) { printf("%zu %zu %zu %zu", sizeof(kore_rope_config), '
                   'sizeof(kore_paged_config), sizeof(kore_paged_batch), sizeof(kore_paged_info)); return 0; }\n')
    exe = tmp_path / "t"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(exe), str(src)], check=True)
    want = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert [C.sizeof(s) for s in (rope.RopeConfig, paged.PagedConfig, paged.BatchStruct, paged.PagedInfo)] == want


@pytest.mark.parametrize("kw,fragment", [
    (dict(rot_dim=0), "rot_dim"), (dict(rot_dim=7), "rot_dim"), (dict(rot_dim=514), "rot_dim"),
    (dict(rot_dim=64, base=0.0), "base"), (dict(rot_dim=64, base=float("inf")), "base"), (dict(rot_dim=64, base=float("nan")), "base"),
    (dict(rot_dim=64, scaling="linear", factor=0.0), "factor"), (dict(rot_dim=64, scaling="linear", factor=float("nan")), "factor"),
    (dict(rot_dim=64, scaling="yarn", factor=0.5, orig_ctx=10), "factor"), (dict(rot_dim=64, scaling="yarn", factor=2.0), "orig_ctx"),
    (dict(rot_dim=64, scaling="yarn", factor=2.0, orig_ctx=10, base=1.0), "base"),
    (dict(rot_dim=64, scaling="yarn", factor=2.0, orig_ctx=10, beta_fast=-1.0), "beta"),
    (dict(rot_dim=64, magnitude=-1.0), "magnitude"), (dict(rot_dim=4, freq_factors=[1.0, 0.0]), "freq_factors[1]"),
    (dict(rot_dim=64, base=1e-30), "frequency"), (dict(rot_dim=64, scaling="linear", factor=1e-38), "frequency 0"),
    (dict(rot_dim=4, base=1.0, freq_factors=[1.0, 2.0 ** -21]), "frequency 1"),
])
def test_rope_refuses(kw, fragment):
    from kore_amd import rope
    with pytest.raises(rope.PagedError) as e:
        rope.Rope(rope.Config(**kw))
    assert e.value.code == rope.KORE_PAGED_E_INVALID and fragment in e.value.message


def test_unknown_names():
    from kore_amd import rope
    for kw in (dict(layout="x"), dict(scaling="x"), dict(freq_factors=np.ones(3))):
        with pytest.raises(ValueError):
            rope.Config(8, **kw)
    with pytest.raises(ValueError):
        rope.type_code("f64")
    cfg = rope.Config(8)
    cfg.struct.layout = 2
    with pytest.raises(rope.PagedError, match="layout"):
        rope.Rope(cfg)
    cfg = rope.Config(8)
    cfg.struct.scaling = 3
    with pytest.raises(rope.PagedError, match="scaling"):
        rope.Rope(cfg)


GOOD = dict(n_layer=1, n_pages=4, page_size=16, n_head=4, n_head_kv=2, head_dim=64)


@pytest.mark.parametrize("kw,code,fragment", [
    (dict(n_layer=0), -1, "non-positive"), (dict(n_pages=-1), -1, "non-positive"), (dict(head_dim=0), -1, "non-positive"),
    (dict(n_head=5), -1, "multiple"), (dict(page_size=8), -1, "page_size"), (dict(page_size=48), -1, "page_size"),
    (dict(page_size=512), -1, "page_size"), (dict(head_dim=60), -3, "head_dim 60"), (dict(head_dim=264), -3, "head_dim 264"),
    (dict(k_pool=4096), -1, "one pool"), (dict(k_pool=4096, v_pool=4100), -1, "aligned"),
    (dict(n_layer=2 ** 20, n_pages=2 ** 30), -1, "overflows"), (dict(n_head=2 ** 17, n_head_kv=2 ** 17), -3, "n_head"),
])
def test_cache_refuses(kw, code, fragment):
    from kore_amd import paged
    with pytest.raises(paged.PagedError) as e:
        paged.PagedKV(**{**GOOD, **kw})
    assert e.value.code == code and fragment in e.value.message


def test_cache_refuses_its_rope():
    from kore_amd import paged, rope
    with pytest.raises(paged.PagedError, match="over head_dim"):
        paged.PagedKV(**GOOD, rope=rope.Config(66))
    with pytest.raises(paged.PagedError, match="base"):
        paged.PagedKV(**GOOD, rope=rope.Config(64, base=-1.0))


def test_null_handles():
    from kore_amd import paged, rope
    L = paged.lib()
    bad = rope.KORE_PAGED_E_INVALID
    assert L.kore_rope_create(None, None) == bad
    h = C.c_void_p()
    assert L.kore_rope_create(C.byref(h), None) == bad and L.kore_paged_create(C.byref(h), None) == bad and not h.value
    assert L.kore_rope_apply_dev(None, 0, 1, 1, 8, None, 8, None, None, 8, 0, None) == bad
    assert L.kore_paged_append_dev(None, 0, None, 0, None, 0, None, 0, None, 0, None, 0, None) == bad
    assert L.kore_paged_attend_dev(None, 0, None, 0, None, 0, None, 0, 0.0, 0, None, None) == bad
    assert L.kore_paged_get_info(None, None) == bad and L.kore_paged_sync(None) == bad and L.kore_rope_sync(None) == bad
    assert L.kore_rope_get_freqs(None, None, None) == bad
    assert L.kore_paged_workspace_bytes(None) == 0
    L.kore_rope_destroy(None)
    L.kore_paged_destroy(None)
    assert L.kore_paged_last_error(None) is not None and L.kore_rope_last_error(None) is not None


@pytest.mark.skipif(os.path.exists("/dev/kfd"), reason="a GPU is present")
def test_create_without_gpu_is_a_hip_error():
    from kore_amd import paged, rope
    for make in (lambda: rope.Rope(rope.Config(64)), lambda: paged.PagedKV(**GOOD, rope=rope.Config(64))):
        with pytest.raises(rope.PagedError) as e:
            make()
        assert e.value.code == rope.KORE_PAGED_E_HIP and e.value.message
