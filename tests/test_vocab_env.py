"""The OpEnvs of the vocabulary operators through the C window, without a GPU: built with
AddressSanitizer and UndefinedBehaviorSanitizer against a recording stand-in for the kernel library
(tests/cpp/test_vocab_env.cc)."""
import os
import subprocess
from concurrent.futures import ThreadPoolExecutor

from tests.test_host_sanitized import DIALECT, ROOT, SAN_FLAGS, SOURCES, write_stub


def test_execute_takes_only_what_the_op_env_was_made_for(tmp_path):
    stub = tmp_path / "stub.cc"
    write_stub(stub, leave_out={"rafhip_device_count", "rafhip_last_error"})
    exe = tmp_path / "test_vocab_env"
    gxx = ["g++", "-std=c++17", "-Wall", *SAN_FLAGS, f"-I{DIALECT}", f"-I{ROOT / 'include'}"]

    def compile_one(src):
        obj = tmp_path / (src.stem + ".o")
        subprocess.run([*gxx, "-c", str(src), "-o", str(obj)], check=True)
        return str(obj)

    sources = [ROOT / "tests" / "cpp" / "test_vocab_env.cc", stub, *[DIALECT / s for s in (*SOURCES, "hip_vocab.cc")]]
    with ThreadPoolExecutor(max_workers=4) as pool:
        subprocess.run([*gxx, *pool.map(compile_one, sources), "-o", str(exe)], check=True)
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=0:verify_asan_link_order=0",
               UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1")
    r = subprocess.run([str(exe)], capture_output=True, text=True, env=env)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-6000:]
    assert "ALL OK" in r.stdout
    assert "runtime error" not in r.stderr and "AddressSanitizer" not in r.stderr and "LeakSanitizer" not in r.stderr
