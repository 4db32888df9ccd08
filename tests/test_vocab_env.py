"""OpEnvs and the C window against recording stand-ins for the kernel library, without a GPU, built with
AddressSanitizer and UndefinedBehaviorSanitizer: what Execute refuses (tests/cpp/test_vocab_env.cc)
the stream that a call runs on (test_call_stream.cc) and the end of stream-ordered memory
(test_memory_release.cc)."""
import os
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from tests.test_host_sanitized import DIALECT, ROOT, SAN_FLAGS, SOURCES, write_stub


@pytest.fixture(scope="module")
def build(tmp_path_factory):
    """Builds a test program against the host layer, whose objects are compiled once, and a kernel library in
    which the functions named in ``own`` are the program's; runs it."""
    out = tmp_path_factory.mktemp("vocab_env")
    gxx = ["g++", "-std=c++17", "-Wall", "-pthread", *SAN_FLAGS, f"-I{DIALECT}", f"-I{ROOT / 'include'}"]

    def compile_one(src):
        obj = out / (src.stem + ".o")
        subprocess.run([*gxx, "-c", str(src), "-o", str(obj)], check=True)
        return str(obj)

    with ThreadPoolExecutor(max_workers=4) as pool:
        layer = list(pool.map(compile_one, [DIALECT / s for s in (*SOURCES, "hip_vocab.cc")]))

    def run(program, own, quiet=True):
        stub = out / f"{program}_stub.cc"
        write_stub(stub, leave_out=own)
        exe = out / program
        subprocess.run([*gxx, compile_one(ROOT / "tests" / "cpp" / f"{program}.cc"), compile_one(stub), *layer, "-o", str(exe)],
                       check=True)
        env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=0:verify_asan_link_order=0",
                   UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1")
        r = subprocess.run([str(exe)], capture_output=True, text=True, env=env, timeout=300)
        assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-6000:]
        assert "ALL OK" in r.stdout
        assert not quiet or not r.stderr
        assert "runtime error" not in r.stderr and "AddressSanitizer" not in r.stderr and "LeakSanitizer" not in r.stderr

    return run


def test_execute_takes_only_what_the_op_env_was_made_for(build):
    build("test_vocab_env", {"rafhip_device_count", "rafhip_last_error"})


def test_streams_of_the_process_and_of_a_call(build):
    build("test_call_stream", {"rafhip_device_count", "rafhip_last_error", "rafhip_sgd"})


def test_stream_ordered_memory_that_outlives_its_stream(build):
    build("test_memory_release", {"rafhip_dev_set", "rafhip_dev_alloc_async", "rafhip_dev_free_async", "rafhip_dev_free"},
          quiet=False)
