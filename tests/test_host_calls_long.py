"""The host code of the long-context calls against a HIP runtime that runs nothing (tests/hip_stub.cpp), on the CPU: refusals,
the device that is current, failed allocations and launches, grids at the largest sizes.  Every scenario is a process of its
own, as in test_host_calls.py.
"""
import ctypes
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

from tests.test_host_calls import DEV, OUT, Engine, P, kernels, stub  # noqa: E402, F401  (stub: the fixture)

FAR = [P((1 << 44) + (i << 40)) for i in range(8)]  # device operands apart from each other


def rotary(e, **kw):
    return ctypes.byref(e._lib.GqaRope(**{**dict(layout=1, base=1e4, factor=1.0), **kw}))


def calls_of(e):
    """Every long-context call of an engine with operands that it takes."""
    c = e.ctx
    return [("gqa_qk_norm_rotary_device", c, 0, FAR[0], 768, 4, None, None, 1e-6, 0, 0, 0, rotary(e), FAR[1], None),
            ("gqa_qk_norm_rotary_step_device", c, FAR[0], 768, None, None, 1e-6, FAR[2], None, rotary(e), FAR[1], None),
            ("gqa_decode_prefix_device", c, FAR[0], 1, 100, None, FAR[2], FAR[1], None, None),
            ("gqa_decode_append_prefix_device", c, FAR[0], FAR[3], FAR[4], FAR[5], 1, 100, FAR[6], FAR[2], FAR[1], FAR[7], None),
            ("gqa_attention_mass_step_device", c, FAR[0], FAR[2], FAR[3], 1.0, FAR[1], None),
            ("gqa_attention_mass_device", c, 0, FAR[0], 20, 80, 100, 0, 1, FAR[3], 0.5, FAR[1], None),
            ("gqa_evict_device", c, FAR[0], FAR[1], 50, 4, 8, FAR[2], FAR[3], FAR[4], None)]


def device_of_calls(stub):
    """The calls work on their context's device whichever is current, and leave that one current."""
    for kv8, room in ((True, 300), (False, 300), (True, 4096), (False, 4096)):
        e = Engine(stub, kv8=kv8, max_seq_len=room)
        for name, *args in calls_of(e):
            e.ok(name, *args)
            log = e.log()
            assert kernels(log), name
            assert all(line[0] == "1" for line in log), (name, log)
            assert e.stub.stub_device() == 0, name


def failures(stub):
    """No memory for the partials: the call says so, launches nothing, and others run; a failed launch is reported once."""
    e = Engine(stub, kv8=False, max_seq_len=4096)  # (short contexts need no partials)
    calls = calls_of(e)
    e.stub.stub_fail_malloc_above(1 << 20)
    name, *args = calls[2]
    assert e.call(name, *args) == e._lib.GQA_ERR_OOM and not kernels(e.log())
    for other, *rest in calls[:2] + calls[4:]:
        e.ok(other, *rest)
    e.stub.stub_fail_malloc_above(1 << 40)
    e.ok(name, *args)
    assert sum(line[1] == "hipMalloc" for line in e.log()) == 1
    for name, *args in calls:
        e.ok(name, *args)
        log = e.log()
        assert not any(line[1] in ("hipMalloc", "hipDeviceSynchronize") for line in log), name
        for at in range(len(kernels(log))):
            e.stub.stub_fail_launch(at)
            assert e.call(name, *args) == e._lib.GQA_ERR_HIP, (name, at)
            assert len(kernels(e.log())) == at + 1
            e.ok("gqa_decode_device", e.ctx, DEV, DEV, OUT, None, None)
            e.log()


def refusals(stub):
    """Operands that are missing, out of range, misaligned or over each other; nothing is launched for them."""
    for kv8, page in ((False, 0), (True, 0), (True, 64)):
        e = Engine(stub, kv8=kv8, page=page)
        L, E = e._lib, e.ctx
        if page:
            e.ok("gqa_paged_reserve", E, 1, 64)
        base = {name: args for name, *args in calls_of(e)}
        kc, vc, cap = P(), P(), ctypes.c_int32()
        e.ok("gqa_cache_pointers", E, ctypes.byref(kc), ctypes.byref(vc), ctypes.byref(cap))
        near = lambda p, n: P(p.value + n)  # noqa: E731
        e.log()

        def refused(name, want, **at):
            args = list(base[name])
            for i, v in at.items():
                args[int(i[1:])] = v
            assert e.call(name, *args) == want, (name, at, kv8, page)
            assert not kernels(e.log()), (name, at)

        for name, pointers in (("gqa_qk_norm_rotary_device", (0, 2, 11, 12)), ("gqa_qk_norm_rotary_step_device", (0, 1, 6, 8, 9)),
                               ("gqa_decode_prefix_device", (0, 1, 5, 6)), ("gqa_decode_append_prefix_device", (0, 1, 2, 3, 4, 8, 9)),
                               ("gqa_attention_mass_step_device", (0, 1, 2, 3, 5)), ("gqa_attention_mass_device", (0, 2, 8, 10)),
                               ("gqa_evict_device", (0, 1, 2, 6, 7, 8))):
            for i in pointers:
                refused(name, L.GQA_ERR_NULL, **{f"a{i}": None})
        R, D = L.GQA_ERR_RANGE, L.GQA_ERR_STREAM_DEST
        name = "gqa_decode_append_prefix_device"
        for b in (-1, 2):
            refused(name, D, a5=b)
        for n in (-1, 301) + ((65,) if page else ()):
            refused(name, R, a6=n)
        for i, n in ((1, 8), (2, 2), (3, 8), (4, 2), (7, 1), (8, 2), (9, 1), (10, 2)):
            refused(name, R, **{f"a{i}": near(FAR[0], n)})
        refused(name, R, a9=kc)
        refused(name, R, a10=near(vc, 4))
        refused("gqa_decode_prefix_device", R, a6=near(kc, 2))
        name = "gqa_attention_mass_step_device"
        for decay in (-0.1, 1.5, float("nan"), float("inf")):
            refused(name, R, a4=decay)
        for i, n in ((1, 8), (2, 2), (3, 1), (5, 2)):
            refused(name, R, **{f"a{i}": near(FAR[0], n)})
        mass_bytes = 2 * 2 * 300 * 4
        for i in (1, 2, 3):
            refused(name, R, a5=base[name][i])
        refused(name, R, a5=near(base[name][3], -mass_bytes + 4))
        refused(name, R, a5=near(vc, 64))
        if not page:  # (rows that are not mapped come first otherwise)
            name = "gqa_attention_mass_device"
            refused(name, D, a1=2)
            refused(name, D, a1=-1)
            for i, v in ((3, 0), (3, 65), (4, -1), (4, 2**31 - 20), (5, 301), (5, -1), (6, -1), (6, 2**31 - 100), (9, 2.0), (10, base[name][2]),
                         (10, base[name][8]), (10, kc), (2, near(FAR[0], 4)), (8, near(FAR[3], 2))):
                refused(name, R, **{f"a{i}": v})
        else:
            refused("gqa_attention_mass_device", R)
            refused("gqa_qk_norm_rotary_device", R)
        name = "gqa_evict_device"
        for keep, sinks, recent in ((0, 0, 0), (301, 0, 0), (50, -1, 0), (50, 0, -1), (50, 25, 26), (50, 2**31 - 1, 2**31 - 1)):
            refused(name, R, a3=keep, a4=sinks, a5=recent)
        mass, lens, new_mass, new_lens, kept = (base[name][i] for i in (1, 2, 6, 7, 8))
        for i in (1, 2, 6, 7, 8):
            refused(name, R, **{f"a{i}": near(base[name][i], 2)})
        for i in (6, 7, 8):
            refused(name, R, **{f"a{i}": near(kc, 16)})
        refused(name, R, a6=near(mass, 4))
        refused(name, R, a6=near(mass, -4))
        refused(name, R, a7=near(lens, 4))
        refused(name, R, a6=lens)
        refused(name, R, a7=mass)
        refused(name, R, a8=mass)
        refused(name, R, a8=near(lens, 4))
        refused(name, R, a8=new_mass)
        refused(name, R, a8=near(new_lens, -4))
        refused(name, R, a7=new_mass)
        e.ok(name, E, mass, lens, 50, 4, 8, mass, lens, kept, None)  # in place


def launches_of_the_largest(stub):
    """Caches, batches and prompts whose work-groups pass 2^24, and the longest prefix."""
    far = [P((1 << 56) + (i << 48)) for i in range(6)]
    e = Engine(stub, batch=1, max_seq_len=1 << 30, page=1 << 16, max_q_len=1 << 20)
    e.ok("gqa_attention_mass_step_device", e.ctx, far[0], far[1], far[2], 1.0, far[3], None)
    e.ok("gqa_evict_device", e.ctx, far[0], far[1], 1 << 29, 4, 8, far[0], far[1], far[2], None)
    e = Engine(stub, batch=1, max_seq_len=1 << 27, max_q_len=1 << 20)
    e.ok("gqa_decode_prefix_device", e.ctx, far[0], 0, 1 << 27, None, far[1], far[2], None, None)
    e.ok("gqa_attention_mass_device", e.ctx, 0, far[0], 1 << 20, 0, 1 << 27, 0, 0, far[1], 1.0, far[2], None)
    assert e.call("gqa_qk_norm_rotary_device", e.ctx, 0, far[0], 768, 1 << 27, None, None, 1e-6, 0, 0, 0, rotary(e), far[1], None) == 0
    many = Engine(stub, batch=1 << 20, n_q_heads=64, n_kv_heads=4, max_seq_len=64, max_q_len=1)
    for name, *args in calls_of(many):
        if "step" in name or "evict" in name:
            args = [64 * 72 if a == 768 else 8 if a == 50 else 2 if a == 4 else 3 if a == 8 else a for a in args]
            many.ok(name, *args)
    many.ok("gqa_decode_prefix_device", many.ctx, far[0], 1, 64, None, far[1], far[2], None, None)
    for line in many.log():
        if line[1] == "launch" and "prefix_merge" in line[2]:
            assert int(line[4]) * int(line[5]) >= 1 << 24  # (2^26 rows, four a work-group)


SCENARIOS = {f.__name__: f for f in (device_of_calls, failures, refusals, launches_of_the_largest)}


@pytest.mark.parametrize("name", SCENARIOS)
def test_scenario(stub, name):  # noqa: F811
    run = subprocess.run([sys.executable, str(Path(__file__).resolve()), str(stub), name], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0, run.stdout + run.stderr


if __name__ == "__main__":
    SCENARIOS[sys.argv[2]](sys.argv[1])
