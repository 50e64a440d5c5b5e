"""The parameters of the cache operators keep the layout that they had before caches of 4 bits: a caller built against
the header of then, which knows no ``bits``, clears its struct and is taken for one of 8 bits."""

import ctypes
import os
import shutil
import subprocess

import pytest

from conftest import REPO
from test_paged_plan_cpu import FAKE, lib  # noqa: F401  (lib: a fixture)

P, I, L, F = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float

BEFORE = {
    "PagedParams": [P, I, *[L] * 5, *[L] * 2, *[P] * 4, L, I, P, L, L, P, P, L, F, I, L, P, L, L, P, I, P, L],
    "KvReadParams": [*[P] * 4, L, I, *[L] * 4, P, L, L, P, P, P, I],
    "KvWriteParams": [P, P, I, *[L] * 3, *[L] * 4, P, *[P] * 4, L, I],
}


def before(name):
    return type(name, (ctypes.Structure,), {"_fields_": [(f"f{i}", t) for i, t in enumerate(BEFORE[name])]})


@pytest.mark.parametrize("name", BEFORE)
def test_the_layout_is_that_of_before(name):
    from low_bit_fake_quant import _lib
    now, then = getattr(_lib, name), before(name)
    assert ctypes.sizeof(now) == ctypes.sizeof(then)
    fields = [f for f, _ in now._fields_ if f != "bits"]
    assert [getattr(now, f).offset for f in fields] == [getattr(then, f"f{i}").offset for i in range(len(fields))]


def test_what_lies_behind_a_struct_of_before_is_not_read(lib):  # noqa: F811
    then = before("PagedParams")

    class Behind(ctypes.Structure):
        _fields_ = [("p", then), ("other", ctypes.c_int * 2)]

    hq, hk, d, cols = 32, 8, 128, 100
    values = [FAKE, 2, 1, hq, hk, d, 1, hq * d, d, FAKE, FAKE, FAKE, FAKE, 4, 6, FAKE, cols, cols, FAKE, FAKE, 1, 0.1, 1, 0,
              FAKE, hq * d, d, None, 0, None, 0]
    b = Behind(then(*values), (ctypes.c_int * 2)(0x55555555, 4))
    need = lib.lbfq_paged_attention_workspace_bytes(ctypes.cast(ctypes.pointer(b.p), ctypes.POINTER(_params())))
    row = hq * (4 * d + 8)
    assert need > 16 and (need - 16) % row == 0


def _params():
    from low_bit_fake_quant import _lib
    return _lib.PagedParams


@pytest.mark.skipif(not shutil.which("gcc"), reason="no C compiler")
def test_the_binding_has_the_headers_layout(tmp_path):
    """Offsets as a C compiler sees them."""
    from low_bit_fake_quant import _lib
    structs = {"PagedParams": "lbfq_paged_params", "KvReadParams": "lbfq_kv_read_params", "KvWriteParams": "lbfq_kv_write_params",
               "KvAppendParams": "lbfq_kv_append_params"}
    lines = [f'printf("%zu\\n", sizeof({c}));' + "".join(f'printf("%zu\\n", offsetof({c}, {f}));' for f, _ in getattr(_lib, n)._fields_)
             for n, c in structs.items()]
    src = tmp_path / "offsets.c"
    src.write_text("#include <stddef.h>\n#include <stdio.h>\n#include \"lbfq.h\"\nint main(void) {\n" + "\n".join(lines) + "\nreturn 0; }\n")
    exe = tmp_path / "offsets"
    subprocess.run(["gcc", "-I", os.path.join(REPO, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for n in structs:
        t = getattr(_lib, n)
        want += [ctypes.sizeof(t)] + [getattr(t, f).offset for f, _ in t._fields_]
    assert got == want
