"""The C entries of scored attention, shared prefixes and block norms under
AddressSanitizer: the refusals of tests/test_scored_host.py against the library that
tests/test_asan_capi.py builds."""
import subprocess
import sys

from .test_asan_capi import ROOT, asan_env, pytestmark  # noqa: F401


def test_refusals_pass_under_asan(asan_env):  # noqa: F811
    _, env = asan_env
    res = subprocess.run([sys.executable, "-m", "pytest", "tests/test_scored_host.py", "-q", "-k",
                          "entries or entry or empty_batches or workspace_sizes",
                          "-p", "no:cacheprovider"], cwd=ROOT, env=env, capture_output=True,
                         text=True, timeout=600)
    out = res.stdout + res.stderr
    assert "AddressSanitizer" not in out, out[-4000:]
    assert res.returncode == 0 and " passed" in out, out[-4000:]
