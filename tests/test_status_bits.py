"""The bits kernels set in a context's status word: read from the sources (a kernel that loses a wait cannot be made to here)."""
import os
import re

from ojas_engine_b200 import _build

SET = re.compile(r"(?:atomicOr\([\w.>-]*status|mbar_wait_\w+\(.*\.status),\s*(0x[0-9a-fA-F]+u?|OJAS_ST_\w+)\)")


def test_every_status_bit_means_one_thing():
    sources = {n: open(os.path.join(_build.CSRC, n)).read() for n in sorted(os.listdir(_build.CSRC)) if n.endswith((".cu", ".cuh"))}
    named = {n: int(v, 16) for text in sources.values() for n, v in re.findall(r"constexpr unsigned (OJAS_ST_\w+) = (0x[0-9a-fA-F]+)u", text)}
    used = [(name, code) for name, text in sources.items() for code in SET.findall(text)]
    assert len(used) > 20
    bits = {}
    for where, code in used:
        value = named[code] if code in named else int(code.rstrip("u"), 16)
        assert value and value & (value - 1) == 0, (where, code)
        bits.setdefault(value, set()).add(code if code in named else where)
    shared = {hex(v): who for v, who in bits.items() if len(who) > 1}
    assert not shared, shared
    ranges = [v for n, v in named.items() if n.endswith("_WAITS")]             # kept for a file's literals
    for where, code in used:
        assert code in named or sum(int(code.rstrip("u"), 16) & m != 0 for m in ranges) == 1, (where, code)
