"""What the long-context calls refuse beyond missing and misplaced operands, against a HIP runtime that runs nothing
(tests/hip_stub.cpp), on the CPU.  Every scenario is a process of its own, as in test_host_calls.py.
"""
import ctypes
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

from tests.test_host_calls import DEV, OUT, Engine, kernels, stub  # noqa: E402, F401  (stub: the fixture)
from tests.test_host_calls_long import calls_of  # noqa: E402


def numerics_of_a_prefix(stub):
    """Decode over a prefix is exact arithmetic alone, as decode: refused under KV260 numerics, in one launch and in two."""
    for room in (300, 4096):
        e = Engine(stub, kv8=False, max_seq_len=room)
        L = e._lib
        calls = [call for call in calls_of(e) if "prefix" in call[0]]
        assert len(calls) == 2
        e.ok("gqa_set_option", e.ctx, L.GQA_OPT_NUMERICS, L.GQA_NUMERICS_KV260)
        for name, *args in calls:
            assert e.call("gqa_decode_device", e.ctx, DEV, DEV, OUT, None, None) == L.GQA_ERR_UNSUPPORTED
            assert e.call(name, *args) == L.GQA_ERR_UNSUPPORTED, (name, room)
            log = e.log()
            assert not kernels(log) and not any(line[1] == "hipMalloc" for line in log), (name, room)
        e.ok("gqa_set_option", e.ctx, L.GQA_OPT_NUMERICS, L.GQA_NUMERICS_EXACT)
        for name, *args in calls:
            e.ok(name, *args)


def magnitude_of_a_rotary_form(stub):
    """What multiplies cosine and sine is an fp32 number: one that fp32 does not hold would make every head NaN."""
    e = Engine(stub)
    L, top = e._lib, (2 - 2.0**-23) * 2.0**127
    out = (ctypes.c_double * 32)()
    for magnitude, want in ((0.0, 0), (1.25, 0), (top, 0), (2.0**128, L.GQA_ERR_RANGE), (1e300, L.GQA_ERR_RANGE), (-1.0, L.GQA_ERR_RANGE),
                            (float("inf"), L.GQA_ERR_RANGE), (float("nan"), L.GQA_ERR_RANGE)):
        form = ctypes.byref(L.GqaRope(layout=1, base=1e4, factor=1.0, magnitude=magnitude))
        assert e.call("gqa_rope_frequencies", form, 64, out, None) == want, magnitude
        for name, *args in calls_of(e):
            if "rotary" in name:
                args[-3] = form
                assert e.call(name, *args) == want, (name, magnitude)
                assert len(kernels(e.log())) == (0 if want else 1), (name, magnitude)


def largest_batches_of_a_prefix(stub):
    """batch * n_kv_heads * max_seq_len up to 2^35, lengths in whole steps of 32 rows; above that refused."""
    for batch, room, want in ((1 << 10, 1 << 22, 0), (1 << 10, (1 << 22) - 31, 0), (1 << 10, (1 << 22) + 1, 0x27), ((1 << 10) + 1, 1 << 22, 0x27)):
        # (of a paged cache: pages for one sequence each, tables for all of their rows)
        e = Engine(stub, page=1 << 16, batch=batch, n_q_heads=8, n_kv_heads=8, max_seq_len=room, max_q_len=1)
        assert e._lib.GQA_ERR_UNSUPPORTED == 0x27
        for name, *args in calls_of(e):
            if "prefix" in name:
                args[2 if name == "gqa_decode_prefix_device" else 5] = 0
                args[3 if name == "gqa_decode_prefix_device" else 6] = 0
                assert e.call(name, *args) == want, (name, batch, room)
                assert bool(kernels(e.log())) == (want == 0)


SCENARIOS = {f.__name__: f for f in (numerics_of_a_prefix, magnitude_of_a_rotary_form, largest_batches_of_a_prefix)}


@pytest.mark.parametrize("name", SCENARIOS)
def test_scenario(stub, name):  # noqa: F811
    run = subprocess.run([sys.executable, str(Path(__file__).resolve()), str(stub), name], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0, run.stdout + run.stderr


if __name__ == "__main__":
    SCENARIOS[sys.argv[2]](sys.argv[1])
