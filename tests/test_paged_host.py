"""The paged-cache operators' boundary, checked without a GPU: the argument
blocks that the Python binding packs are the header's structs, and a call
without a device handle is refused."""
import ctypes
import re
import subprocess
from pathlib import Path

import pytest

pytest.importorskip("torch")
from bnn_b200 import _lib, accel, paged  # noqa: E402

ROOT = Path(__file__).resolve().parents[1]


def test_packed_blocks_match_the_header(tmp_path):
    text = (ROOT / "include" / "bnn_b200_paged.h").read_text()
    # every member is eight bytes wide, in the order the binding packs them
    members = {}
    for body, name in re.findall(r"typedef struct \{(.*?)\} (BNN_Paged\w+);", text, re.S):
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        members[name] = [m.strip().lstrip("*").split("[")[0] for line in body.split(";") if line.strip()
                         for m in line.strip().split(None, 1)[1].replace("void*", "").replace("float*", "").replace("int32_t*", "").split(",")]
    src = tmp_path / "probe.c"
    lines = "\n".join(
        f'printf("{n}.{m} %zu %zu\\n", offsetof({n}, {m.split()[-1].lstrip("*")}), sizeof((({n}*)0)->{m.split()[-1].lstrip("*")}));'
        for n, ms in members.items() for m in ms)
    sizes = "\n".join(f'printf("{n} %zu\\n", sizeof({n}));' for n in members)
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "bnn_b200_paged.h"\nint main(void) {{\n{lines}\n{sizes}\nreturn 0; }}\n')
    exe = tmp_path / "probe"
    subprocess.run(["gcc", "-std=c11", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split("\n")
    got = dict(line.split(" ", 1) for line in out if line)
    for name, size in paged._sizes().items():
        assert int(got[name]) == size
    at = {}
    for key, value in got.items():
        if "." in key:
            name, member = key.split(".")
            offset, width = map(int, value.split())
            assert offset == at.get(name, 0), key  # no gaps
            assert width == (int(got["BNN_PagedCache"]) if member == "cache" else 8), key
            at[name] = offset + width


@pytest.mark.parametrize("name", ["bnn_b200_paged_append", "bnn_b200_paged_attention"])
def test_no_handle_is_refused(name):
    fn = getattr(_lib.load(), name)
    fn.restype = ctypes.c_int
    fn.argtypes = [ctypes.c_void_p, ctypes.c_char_p, ctypes.c_void_p]
    assert fn(None, bytes(512), None) == accel.EINVAL
    sync = _lib.load().bnn_b200_paged_sync
    sync.restype = ctypes.c_int
    sync.argtypes = [ctypes.c_void_p, ctypes.c_void_p]
    assert sync(None, None) == accel.EINVAL
