"""The binding resolves an op as Plugin.resolve does: the row with the highest priority of both tables. A stand-in for the
loader's table, put in front of the library's, declares a row of higher priority that answers with a status."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent

TABLE = """
#include "rad_abi.h"
#include "rad_plugin.h"
static int answer(const RadArgs*, RadStream) { return RAD_E_UNSUPPORTED; }
static RadKernelInfo make(const char* name, int priority) {
    RadKernelInfo k = {};
    k.name = name; k.op = "quant_token_i8"; k.priority = priority; k.launch = answer;
    return k;
}
extern "C" const RadKernelInfo* rad_kernel_at(int i) {
    static const RadKernelInfo rows[2] = {make("below", 1), make("stand-in", PRIORITY)};
    return i >= 0 && i < 2 ? &rows[i] : nullptr;
}
"""
CODE = """
import torch
from libr3d_b200 import ops
try:
    ops.quant_token_i8(torch.ones(2, 16, device="cuda"))
    print("extension row")
except ops.RowRefused as e:
    print(e)
"""


@pytest.mark.parametrize("priority,want", [(5000, "row stand-in returned"), (1000, "row stand-in returned"), (999, "extension row")])
def test_the_row_of_highest_priority_serves_the_call(tmp_path, priority, want):
    (tmp_path / "table.cpp").write_text(TABLE)
    so = tmp_path / "table.so"
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", f"-DPRIORITY={priority}", "-I", str(ROOT / "include"), str(tmp_path / "table.cpp"), "-o", str(so)], check=True)
    r = subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, env=os.environ | {"LD_PRELOAD": str(so)}, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.startswith(want), r.stdout + r.stderr[-2000:]
