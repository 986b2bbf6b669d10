"""The list planner (csrc/plan.cpp) built by itself with g++, for planning against buffers of stated sizes: b200q_plan takes
buffers of any size, and a context needs a GPU."""
import ctypes
import os
import subprocess

import numpy as np

from conftest import ROOT

SOURCE = r"""
#include "plan.h"
using namespace b200q;
extern "C" int plan_with(const uint32_t *cmds, unsigned n, size_t act_floats, size_t state_rows, size_t kv_bytes) {
    Limits lim;
    lim.act_floats = act_floats;
    lim.state_rows = state_rows;
    lim.kv_bytes = kv_bytes;
    return plan_list(cmds, n, lim).status;
}
"""


def build(folder):
    """plan(cmds, act_floats, state_rows, kv_bytes) -> status, from a library built in `folder`."""
    csrc = os.path.join(ROOT, "fpga-llama-gguf_b200", "csrc")
    src, out = os.path.join(folder, "plan_with.cpp"), os.path.join(folder, "plan_with.so")
    with open(src, "w") as f:
        f.write(SOURCE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-fPIC", "-shared", "-I", csrc, src, os.path.join(csrc, "plan.cpp"), "-o", out], check=True, timeout=300)
    f = ctypes.CDLL(out).plan_with
    f.argtypes = [ctypes.c_void_p, ctypes.c_uint, ctypes.c_size_t, ctypes.c_size_t, ctypes.c_size_t]

    def plan(cmds, act_floats=1 << 22, state_rows=1 << 10, kv_bytes=1 << 20):
        c = np.ascontiguousarray(cmds, np.uint32)
        return f(c.ctypes.data, len(c) // 8, act_floats, state_rows, kv_bytes)

    return plan
