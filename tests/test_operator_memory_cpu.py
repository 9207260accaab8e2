"""Operators' host code when memory runs out: an error or a slower call, no
exception through the C interface.  No kernel is launched.  CPU only."""
from __future__ import annotations

import os
import subprocess
import sys
import textwrap

from conftest import ROOT


def test_descriptor_caches_without_memory(tmp_path):
    exe = str(tmp_path / "tmap_memory_check")
    cuda_inc = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include")
    csrc = os.path.join(ROOT, "paged-speculative-engine_b200", "csrc")
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{csrc}", f"-I{cuda_inc}",
                    os.path.join(ROOT, "tests", "native", "tmap_memory_check.cpp"), "-o", exe], check=True)
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.strip() == "OK", out.stdout + out.stderr


def test_work_list_without_memory():
    """A list of 100 million items in an address space that cannot hold it."""
    child = textwrap.dedent("""
        import ctypes, resource, sys
        import numpy as np
        from pse import _native
        lib = _native.load(require_cuda=False)
        n, lens = ctypes.c_int64(0), np.asarray([200_000_000], dtype=np.int32)
        plan = np.zeros(0, dtype=np.int32)
        now = int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize()
        resource.setrlimit(resource.RLIMIT_AS, (now + (1 << 30), resource.RLIM_INFINITY))
        # (the items are collected before the list is written: 2.4 GB that are refused)
        rc = lib.pse_prompt_plan(lens.ctypes.data, 1, 128, 1, 148, plan.ctypes.data, 1 << 40, ctypes.addressof(n))
        print("code", rc, n.value)
    """)
    env = dict(os.environ, PYTHONPATH=os.path.join(ROOT, "paged-speculative-engine_b200"))
    out = subprocess.run([sys.executable, "-c", child], capture_output=True, text=True, env=env)
    assert out.stdout.split() == ["code", "10001", str(148 + 4 + 4 * 100_000_000)], out.stdout + out.stderr
