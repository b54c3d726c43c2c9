"""CPU tests of the recurrent-block operators' C structs: the ctypes layouts and
the packed forms the helpers fill equal the C compiler's."""
import ctypes
import os
import struct
import subprocess

import pytest

import mamba_b200 as mb

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {
    "MambaRecurrenceArgs": (mb.MambaRecurrenceArgs, mb._RECURRENCE_ARGS),
    "MambaRecurrenceGrads": (mb.MambaRecurrenceGrads, mb._RECURRENCE_GRADS),
    "MambaBlockNormArgs": (mb.MambaBlockNormArgs, mb._BLOCK_NORM_ARGS),
    "MambaBlockNormGrads": (mb.MambaBlockNormGrads, mb._BLOCK_NORM_GRADS),
}


def c_name(field):
    return field.rstrip("_")


@pytest.fixture(scope="module")
def layouts(tmp_path_factory):
    lines = []
    for name, (cls, _) in STRUCTS.items():
        lines.append('printf("%s sizeof %%zu\\n", sizeof(%s));' % (name, name))
        for field, *_ in cls._fields_:
            lines.append('printf("%s %s %%zu\\n", offsetof(%s, %s));' % (name, field, name, c_name(field)))
    tmp = tmp_path_factory.mktemp("layout")
    src, exe = str(tmp / "probe.c"), str(tmp / "probe")
    with open(src, "w") as f:
        f.write("#include <stddef.h>\n#include <stdio.h>\n#include \"mamba.h\"\nint main(void) {\n%s\nreturn 0;\n}\n"
                % "\n".join(lines))
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), src, "-o", exe],
                   check=True)
    out = subprocess.run([exe], capture_output=True, text=True, check=True).stdout
    return {tuple(line.split()[:2]): int(line.split()[2]) for line in out.splitlines()}


@pytest.mark.parametrize("name", sorted(STRUCTS))
def test_ctypes_layout_is_the_header_s(layouts, name):
    cls, packed = STRUCTS[name]
    assert ctypes.sizeof(cls) == layouts[name, "sizeof"] == packed.size
    for field, *_ in cls._fields_:
        assert getattr(cls, field).offset == layouts[name, field], field


@pytest.mark.parametrize("name", sorted(STRUCTS))
def test_packed_values_land_in_their_fields(name):
    cls, packed = STRUCTS[name]
    codes = struct.unpack  # every value distinct, in the order the struct lists them
    n = len(codes(packed.format, bytes(packed.size)))
    s = cls.from_buffer_copy(packed.pack(*range(1, n + 1)))
    got = []
    for field, *_ in cls._fields_:
        if field.startswith(("reserved", "pad")):
            continue
        v = getattr(s, field)
        got += list(v) if isinstance(v, ctypes.Array) else [v]
    assert got == list(range(1, n + 1))
