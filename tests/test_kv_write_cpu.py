"""CPU test of what a write of new rows launches: up to 2048 rows every workgroup looks at
the whole call, beyond that one workgroup before them (over the stand-in runtime of
test_host_calls.py)."""
import ctypes

import g4hip
from test_host_calls import Program, hip  # noqa: F401  (the fixture)
from test_kv_cpu import struct


def test_the_check_is_a_launch_of_its_own_for_many_rows(hip):  # noqa: F811
    with Program(hip) as p:
        s, rope = struct(), g4hip._RopeStruct(4096, 64, 0, 1.0)
        stream = p.stream()
        for rows, check in ((1, False), (2048, False), (2049, True), (100000, True)):
            for capturing in (0, 1):  # recorded as well: it needs no workspace
                p.use(stream)
                hip.stub_capture(stream, capturing)
                before = len(p.log())
                assert hip.g4_kv_rope_write_dev(p.ctx, ctypes.addressof(s), 1, ctypes.addressof(rope), 1 << 20, 1 << 20,
                                                4096, 8192, 8, 3, 4096, 4096, rows) == 0
                names = [line[1] for line in p.log()[before:] if line[0] == "launch"]
                assert ["k_kv_write_check" in n for n in names] == ([True, False] if check else [False])
                assert all("k_kv_write" in n for n in names)
                hip.stub_capture(stream, 0)
        p.use(None)
