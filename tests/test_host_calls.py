"""The engine's host code against a HIP runtime that runs nothing (tests/hip_stub.cpp): which device is current where
something is launched or allocated, what follows a failed allocation or launch, and whether launches keep to the
runtime's limits.  On the CPU; every scenario is a process of its own.
"""
import ctypes
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
P = ctypes.c_void_p


class Engine:
    """libgqa.so over the stub, and an E4M3 context on device 1 while device 0 is current."""

    def __init__(self, stub, kv8=True, page=0, **cfg):
        sys.path.insert(0, str(ROOT))
        self.stub = ctypes.CDLL(stub, mode=ctypes.RTLD_GLOBAL)
        self.stub.stub_take_log.restype = ctypes.c_char_p
        self.stub.stub_fail_malloc_above.argtypes = [ctypes.c_size_t]
        from lara_amd import _lib

        self._lib, self.lib = _lib, _lib.lib()
        kw = dict(batch=2, n_q_heads=8, n_kv_heads=2, head_dim=64, max_seq_len=300, max_q_len=64, scale=0.0, device=1)
        kw.update(cfg)
        self.cfg = kw
        c, self.ctx = _lib.GqaConfig(**kw), P()
        if kv8:
            n_pages = kw["batch"] * -(-kw["max_seq_len"] // page) if page else 0
            self.ok("gqa_create_kv8", ctypes.byref(c), page, n_pages, 1, ctypes.byref(self.ctx))
        else:
            self.ok("gqa_create", ctypes.byref(c), ctypes.byref(self.ctx))
        self.stub.hipSetDevice(0)
        self.log()

    def call(self, name, *args):
        return getattr(self.lib, name)(*args)

    def ok(self, name, *args):
        rc = self.call(name, *args)
        assert rc == 0, (name, rc)

    def log(self):
        return [line.split() for line in self.stub.stub_take_log().decode().splitlines()]


DEV = P(0x10000)  # a device operand: the stub's kernels read nothing
OUT = P(0x90000000)


def kernels(log):
    return [line[2] for line in log if line[1] == "launch"]


# ---- scenarios -------------------------------------------------------------------------------------------

def device_of_calls(stub):
    """Device entry points of an E4M3 context work on its device whichever is current, and leave that one current."""
    e = Engine(stub)
    c, graph, cfg = e.ctx, P(), e._lib.GqaConfig(**e.cfg)
    e.ok("gqa_graph_capture_decode_append", c, DEV, DEV, DEV, DEV, DEV, OUT, None, ctypes.byref(graph))
    assert e.stub.stub_device() == 0
    calls = [
        ("gqa_load_kv_device", c, 0, 0, 100, DEV, DEV, None),
        ("gqa_append_kv_device", c, DEV, DEV, DEV, None),
        ("gqa_read_kv_device", c, 0, 0, 100, DEV, OUT, None),
        ("gqa_decode_device", c, DEV, DEV, OUT, None, None),
        ("gqa_decode_append_device", c, DEV, DEV, DEV, DEV, DEV, OUT, None, None),
        ("gqa_prefill_device", c, 0, DEV, 20, 80, 100, 0, 1, OUT, None, None),
        ("gqa_prefill_append_device", c, 0, DEV, DEV, DEV, 20, 20, 80, 100, 0, 1, OUT, None, None),
        ("gqa_qk_norm_rope_device", c, 0, DEV, 768, 4, None, None, 1e-6, 0, 0, 0, 1e4, OUT, None),
        ("gqa_qk_norm_rope_step_device", c, DEV, 768, None, None, 1e-6, DEV, None, 1e4, OUT, None),
        ("gqa_layer_qkv_device", c, 0, DEV, 4, 1024, DEV, DEV, DEV, None, 1e-5, 0, 0, 0, 1, OUT, None),
        ("gqa_w4_pack_device", c, DEV, DEV, 16, 128, 128, OUT, P(0xA0000000), None),
        ("gqa_w4_unpack_device", c, DEV, DEV, 16, 128, 128, OUT, None),
        ("gqa_w4_project_device", c, DEV, 3, 128, DEV, DEV, 128, 16, None, 1e-5, OUT, 16, None),
        ("gqa_graph_launch", graph, None),
        ("gqa_decode_append_noalloc", ctypes.byref(cfg), DEV, DEV, 320, DEV, DEV, DEV, DEV, DEV, OUT, None, None),
    ]
    for name, *args in calls:
        e.ok(name, *args)
        log = e.log()
        assert kernels(log), name
        assert all(line[0] == "1" for line in log), (name, log)
        assert e.stub.stub_device() == 0, name
    # a longer history grows the workspace: what it frees and waits for is on that device too
    e = Engine(stub, max_seq_len=1 << 15)
    for kv_len in (100, 1 << 15):
        e.ok("gqa_prefill_device", e.ctx, 0, DEV, 20, kv_len - 20, kv_len, 0, 1, OUT, None, None)
        log = e.log()
        assert any(line[1] == "hipMalloc" for line in log) and all(line[0] == "1" for line in log), log
        assert e.stub.stub_device() == 0
    assert {"hipDeviceSynchronize", "hipFree"} <= {line[1] for line in log}


def workspace_of_the_exact_size(stub):
    """Where the workspace rounded up cannot be had, calls go on with one of the size they need, and the failed allocation
    is not reported by a launch behind it."""
    e = Engine(stub, max_seq_len=1 << 16, max_q_len=1000)
    rows = 40000  # K and V in bf16: 2 heads * 64 values * 2 * 2 bytes a row, 20.5 MB; rounded up 32 MiB
    e.stub.stub_fail_malloc_above(24 << 20)
    e.ok("gqa_prefill_device", e.ctx, 0, DEV, 20, rows - 20, rows, 0, 1, OUT, None, None)
    log = e.log()
    assert [int(line[2]) for line in log if line[1] == "hipMalloc"] == [32 << 20, rows * 512] and len(kernels(log)) >= 2
    # nothing to be had at all: the call says so, and the next one that needs no more than is there runs
    e.stub.stub_fail_malloc_above(0)
    assert e.call("gqa_prefill_device", e.ctx, 0, DEV, 20, 60000, 60020, 0, 1, OUT, None, None) == e._lib.GQA_ERR_OOM
    e.ok("gqa_decode_device", e.ctx, DEV, DEV, OUT, None, None)
    e.stub.stub_fail_malloc_above(1 << 40)
    e.ok("gqa_prefill_device", e.ctx, 0, DEV, 20, 60000, 60020, 0, 1, OUT, None, None)
    # the layer stage's buffer of projected rows likewise
    e.stub.stub_fail_malloc_above(0)
    assert e.call("gqa_layer_qkv_device", e.ctx, 0, DEV, 1000, 512, DEV, DEV, DEV, None, 1e-5, 0, 0, 0, 1, OUT, None) == e._lib.GQA_ERR_OOM
    e.ok("gqa_decode_device", e.ctx, DEV, DEV, OUT, None, None)
    # a context that cannot be had leaves the others as they are
    cfg, other = e._lib.GqaConfig(**e.cfg), P()
    e.stub.stub_fail_malloc_above(1 << 20)
    assert e.call("gqa_create_kv8", ctypes.byref(cfg), 0, 0, 1, ctypes.byref(other)) == e._lib.GQA_ERR_OOM and not other
    e.ok("gqa_decode_device", e.ctx, DEV, DEV, OUT, None, None)


def workspace_after_a_failed_launch(stub):
    """Whichever launch of a call fails, the next use of the workspace on another stream waits for what the call had
    launched before."""
    e = Engine(stub)
    host = (ctypes.c_uint16 * (2 * 300 * 64))()
    other = P(0x777000)
    calls = [
        ("gqa_prefill_device", e.ctx, 0, DEV, 20, 80, 100, 0, 1, OUT, None, None),
        ("gqa_prefill_append_device", e.ctx, 0, DEV, DEV, DEV, 20, 20, 80, 100, 0, 1, OUT, None, None),
        ("gqa_layer_qkv_device", e.ctx, 0, DEV, 4, 1024, DEV, DEV, DEV, None, 1e-5, 0, 0, 0, 1, OUT, None),
        ("gqa_load_kv", e.ctx, 0, 0, 300, host, host),
        ("gqa_read_kv", e.ctx, 0, 0, 300, host, host),
    ]
    for name, *args in calls:
        e.log()
        e.ok(name, *args)
        launches = len(kernels(e.log()))
        assert launches >= 1, name
        for at in range(launches):
            e.stub.stub_fail_launch(at)
            assert e.call(name, *args) == e._lib.GQA_ERR_HIP, (name, at)
            log = e.log()
            assert len(kernels(log)) == at + 1
            failed = max(i for i, line in enumerate(log) if line[1] == "launch")
            marks = [line[2] for line in log[failed:] if line[1] == "hipEventRecord"]
            e.ok("gqa_prefill_device", e.ctx, 0, DEV, 20, 80, 100, 0, 1, OUT, None, other)
            log = e.log()
            first = min(i for i, line in enumerate(log) if line[1] == "launch")
            waited = [line[2] for line in log[:first] if line[1] == "hipStreamWaitEvent"]
            assert len(waited) == 1 and waited[0] in marks, (name, at, marks, waited)


def launches_of_the_largest_matrices(stub):
    """Packing and unpacking 4-bit matrices up to the documented sizes keeps to the runtime's limit of 2^32 - 1 work-items a
    dimension, with a work-item for every 8 codes."""
    e = Engine(stub)
    far = [P(i << 40) for i in range(1, 5)]
    for rows, hidden, group in ((1 << 20, 1 << 16, 128), (1 << 20, 1 << 16, 32), ((1 << 19) + 1, 1 << 16, 64), (1, 32, 32), (1000, 4096, 128)):
        threads = -(-rows // 16) * -(-hidden // 128) * 256
        e.ok("gqa_w4_pack_device", e.ctx, far[0], far[1], rows, hidden, group, far[2], far[3], None)
        e.ok("gqa_w4_unpack_device", e.ctx, far[2], far[3], rows, hidden, group, far[0], None)
        for line in e.log():
            x, y, _, block = (int(n) for n in line[4:8])
            assert threads <= x * y * block < threads + (block if y == 1 else block << 16)


def launches_of_the_longest_caches(stub):
    """Rows written and read back, heads and the decode merge at sizes whose work-items pass 2^32."""
    n = 1 << 28
    e = Engine(stub, batch=1, max_seq_len=n)
    far = [P((1 << 56) + (i << 48)) for i in range(4)]

    def blocks(kernel, least):
        (line,) = [line for line in e.log() if line[1] == "launch" and kernel in line[2]]
        x, y = int(line[4]), int(line[5])
        assert least <= x * y < least + (1 << 16), line

    e.ok("gqa_load_kv_device", e.ctx, 0, 0, n, far[0], far[1], None)
    blocks("kv8_write", 2 * n * 8 // 256)
    e.ok("gqa_read_kv_device", e.ctx, 0, 0, n, far[0], far[1], None)
    blocks("kv_read", 2 * n * 8 // 256)
    e.ok("gqa_prefill_device", e.ctx, 0, far[0], 20, n - 20, n, 0, 1, far[2], None, None)
    blocks("kv_read", 2 * n * 8 // 256)
    e.ok("gqa_qk_norm_rope_device", e.ctx, 0, far[0], 768, n, None, None, 1e-6, 0, 0, 0, 1e4, far[2], None)
    blocks("qk_norm_rope", n // 2)  # (two tokens a work-group)
    bf16 = Engine(stub, kv8=False, batch=1, n_q_heads=1, n_kv_heads=1, head_dim=128, max_seq_len=1 << 24)
    bf16.ok("gqa_read_kv_device", bf16.ctx, 0, 0, 1 << 24, far[0], far[1], None)
    bf16.ok("gqa_qk_norm_rope_device", bf16.ctx, 0, far[0], 384, 1 << 24, None, None, 1e-6, 0, 0, 0, 1e4, far[2], None)
    many = Engine(stub, batch=1 << 20, n_q_heads=64, n_kv_heads=4, max_seq_len=64, max_q_len=1)
    many.ok("gqa_decode_device", many.ctx, far[0], far[1], far[2], None, None)
    assert "merge" in kernels(many.log())[-1]
    many.ok("gqa_qk_norm_rope_step_device", many.ctx, far[0], 72 * 64, None, None, 1e-6, far[1], None, 1e4, far[2], None)
    many.ok("gqa_append_kv_device", many.ctx, far[0], far[1], far[2], None)


def decode_pieces_of_the_longest_caches(stub):
    """GQA_OPT_DECODE_CHUNK up to its largest value in a context of 2^30 rows: a piece of 2^30 keys holds them all."""
    e = Engine(stub, page=1 << 16, batch=1, max_seq_len=1 << 30, max_q_len=1)
    e.lib.gqa_set_option.argtypes = [P, ctypes.c_int32, ctypes.c_int64]
    for chunk, grid in ((1 << 30, 1), ((1 << 30) + 64, 1), ((1 << 29) + 64, 1), (1 << 29, 2), ((1 << 28) + 64, 2)):
        e.ok("gqa_set_option", e.ctx, e._lib.GQA_OPT_DECODE_CHUNK, chunk)
        e.ok("gqa_decode_device", e.ctx, DEV, DEV, OUT, None, None)
        (line, *_) = [line for line in e.log() if line[1] == "launch"]
        assert "decode_kv8_kernel" in line[2] and int(line[4]) == grid, (chunk, line)


def contexts_past_any_memory(stub):
    """Sizes whose tables or pools no machine holds, or whose bytes pass 64 bits, are refused as out of memory; neither an
    exception nor a small allocation comes of them."""
    e = Engine(stub)
    tables = dict(e.cfg, batch=1 << 16, max_seq_len=1 << 30)
    pools = dict(e.cfg, batch=1 << 21, n_q_heads=1 << 13, n_kv_heads=1 << 13, max_seq_len=1 << 30)  # 2^64 rows
    cfg, ctx = e._lib.GqaConfig(**tables), P()
    for create, *args in (("gqa_create_kv8", 64, 100, 1), ("gqa_create_paged", 64, 100), ("gqa_create_paged_layers", 64, 100, 2)):
        assert e.call(create, ctypes.byref(cfg), *args, ctypes.byref(ctx)) == e._lib.GQA_ERR_OOM and not ctx, create
    cfg = e._lib.GqaConfig(**pools)
    for create, *args in (("gqa_create_kv8", 0, 0, 1), ("gqa_create",), ("gqa_create_kv8", 64, (1 << 31) - 1, 1024)):
        assert e.call(create, ctypes.byref(cfg), *args, ctypes.byref(ctx)) == e._lib.GQA_ERR_OOM and not ctx, create
    cfg = e._lib.GqaConfig(**dict(e.cfg, batch=1 << 21, n_q_heads=1 << 13, n_kv_heads=1 << 9, max_seq_len=1 << 30))  # 2^64 bytes of partials
    assert e.call("gqa_create_paged", ctypes.byref(cfg), 1 << 16, 100, ctypes.byref(ctx)) == e._lib.GQA_ERR_OOM and not ctx
    assert not any(line[1] == "hipMalloc" and int(line[2]) < 1 << 20 for line in e.log())
    e.ok("gqa_decode_device", e.ctx, DEV, DEV, OUT, None, None)


SCENARIOS = {f.__name__: f for f in (device_of_calls, workspace_of_the_exact_size, workspace_after_a_failed_launch,
                                     launches_of_the_largest_matrices, launches_of_the_longest_caches,
                                     decode_pieces_of_the_longest_caches, contexts_past_any_memory)}


@pytest.fixture(scope="module")
def stub(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    so = tmp_path_factory.mktemp("hip_stub") / "libhip_stub.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__",
                    "-I/opt/rocm/include", str(ROOT / "tests" / "hip_stub.cpp"), "-o", str(so)], check=True, timeout=120)
    return so


@pytest.mark.parametrize("name", SCENARIOS)
def test_scenario(stub, name):
    run = subprocess.run([sys.executable, str(Path(__file__).resolve()), str(stub), name], capture_output=True, text=True,
                         timeout=60)
    assert run.returncode == 0, run.stdout + run.stderr


if __name__ == "__main__":
    SCENARIOS[sys.argv[2]](sys.argv[1])
