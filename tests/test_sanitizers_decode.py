"""AddressSanitizer / UndefinedBehaviorSanitizer build of the host code of the
paged decoding entry points, run on the CPU (see test_sanitizers.py, whose
flags it takes)."""
import concurrent.futures
import os
import shutil
import subprocess
import tempfile

import pytest

from tests.conftest import ROOT, gpu_available
from tests.test_sanitizers import SAN

pytestmark = pytest.mark.slow

SOURCES = ["capi_decode.cpp", "rope.hip", "paged_cache.hip", "paged_attn.hip", "paged_attn_latent.hip"]


def test_decode_host_code_under_asan_ubsan():
    from dsa_triton_ascend_amd import build_lib as bl
    try:
        hipcc = bl.hipcc()
    except RuntimeError:
        pytest.skip("hipcc not available")
    if gpu_available():
        pytest.skip("the sweep calls entry points with dummy pointers; it only runs without a GPU")
    work = tempfile.mkdtemp(prefix="dsa_san_")
    try:
        def compile_one(src):
            obj = os.path.join(work, os.path.basename(src) + ".o")
            path = src if os.path.isabs(src) else os.path.join(bl.CSRC, src)
            lang = ["-x", "hip"] if src.endswith(".cpp") else []
            cmd = ([hipcc] + lang + bl.common_flags() + bl.PER_SOURCE_FLAGS.get(src, []) + SAN + ["-c", path, "-o", obj])
            r = subprocess.run(cmd, capture_output=True, text=True)
            return src, obj, r.returncode, r.stdout + r.stderr

        driver = os.path.join(ROOT, "tests", "sanitize", "capi_check_decode.cpp")
        with concurrent.futures.ThreadPoolExecutor(max_workers=6) as ex:
            results = list(ex.map(compile_one, SOURCES + [driver]))
        for src, _, rc, log in results:
            assert rc == 0, f"sanitized build of {src} failed:\n{log[-3000:]}"
        exe = os.path.join(work, "capi_check_decode")
        cmd = [hipcc, f"--offload-arch={bl.ARCH}"] + SAN + [o for _, o, _, _ in results] + ["-o", exe, "-lpthread"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        assert r.returncode == 0, f"link failed:\n{(r.stdout + r.stderr)[-3000:]}"
        env = dict(os.environ)
        env["ASAN_OPTIONS"] = "detect_leaks=0:abort_on_error=0:halt_on_error=1"
        env["UBSAN_OPTIONS"] = "halt_on_error=1:print_stacktrace=1"
        r = subprocess.run([exe], capture_output=True, text=True, env=env, timeout=600)
        assert r.returncode == 0, f"sweep failed (rc {r.returncode}):\n{(r.stdout + r.stderr)[-5000:]}"
        assert "OK" in r.stdout or "SKIP" in r.stdout
        print(r.stdout.strip())
    finally:
        shutil.rmtree(work, ignore_errors=True)
