"""CPU: how a call of the row operators is shared out goes by the current device alone: not by the thread that asks, nor by
what that thread called before. The device is a stand-in for the HIP runtime's two queries (in a process of its own); no call
here gets as far as a launch. And what sizes are refused."""
from __future__ import annotations

import ctypes
import json
import subprocess
import sys
from pathlib import Path

import pytest

from test_rows_abi import forward, params, refused

ROOT = Path(__file__).resolve().parent.parent

SHIM = r"""
#include <hip/hip_runtime_api.h>
#include <cstring>
extern "C" hipError_t hipGetDevice(int * d) { *d = 0; return hipSuccess; }
extern "C" hipError_t hipGetDeviceProperties(hipDeviceProp_t * p, int) {
    std::memset(p, 0, sizeof(*p));
    std::strcpy(p->gcnArchName, "gfx950:sramecc+:xnack-");
    p->multiProcessorCount = CUS;
    return hipSuccess;
}
"""

CHILD = r"""
import ctypes, json, sys, threading
shim, lib, before = sys.argv[1:]
ctypes.CDLL(shim, ctypes.RTLD_GLOBAL)
L = ctypes.CDLL(lib)
L.nxg_last_error.restype = ctypes.c_char_p
for f in ("nxg_attention_rows_workspace_bytes", "nxg_attention_rows_backward_workspace_bytes"):
    getattr(L, f).restype = ctypes.c_int64
i32, P = ctypes.c_int32, ctypes.c_void_p


class Params(ctypes.Structure):
    _fields_ = [(n, i32) for n in ("type", "n_head", "n_kv_head", "head_dim", "T_q", "T_k", "n_seqs")] + [("cu_q", P), ("cu_k", P), ("left", i32), ("right", i32),
                ("scale", ctypes.c_float)]


class Rows(ctypes.Structure):
    _fields_ = [("data", P), ("ts", ctypes.c_int64), ("hs", ctypes.c_int64)]


def params(T_q, T_k):
    return Params(30, 8, 8, 64, T_q, T_k, 1, 1 << 20, 1 << 20, -1, -1, 0.125)


def sizes():
    few, long = params(1, 65536), params(2000, 2000)
    n = int(L.nxg_attention_rows_backward_workspace_bytes(ctypes.byref(long)))
    # what the call itself asks for, from its refusal of any less
    at = [ctypes.byref(Rows((2 + k) << 20, 512, 64)) for k in range(8)]
    rc = L.nxg_attention_rows_backward(ctypes.byref(long), at[0], at[1], at[2], at[3], at[4], P(1 << 20), at[5], at[6], at[7], P(1 << 20),
                                       ctypes.c_int64(16), None)
    return [int(L.nxg_attention_rows_workspace_bytes(ctypes.byref(few))), n, rc, L.nxg_last_error().decode()]


def in_thread(f):
    got = []
    t = threading.Thread(target=lambda: got.append(f()))
    t.start()
    t.join()
    return got[0]


res = []
if before == "new":
    res.append(in_thread(sizes))
res.append([L.nxg_init(), sizes()][1])
res.append(in_thread(sizes))
res.append(sizes())
print(json.dumps(res))
"""


def sizes_of(tmp_path, nxg, cus, before):
    src, shim = tmp_path / f"shim{cus}.cpp", tmp_path / f"shim{cus}.so"
    src.write_text(SHIM)
    rocm = "/opt/rocm/include"
    if not Path(rocm, "hip", "hip_runtime_api.h").exists():
        pytest.skip("no HIP headers")
    subprocess.run(["g++", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", f"-DCUS={cus}", f"-I{rocm}", str(src), "-o", str(shim)], check=True)
    r = subprocess.run([sys.executable, "-c", CHILD, str(shim), str(nxg.LIB_PATH), before], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    return json.loads(r.stdout)


@pytest.mark.parametrize("before", ["new", "known"])
def test_plans_go_by_the_device(tmp_path, nxg, before):
    got = {}
    for cus in (32, 256):
        res = sizes_of(tmp_path, nxg, cus, before)
        forward, backward, rc, refusal = res[0]
        assert all(r == res[0] for r in res), (cus, res)
        assert rc == nxg.NXG_EINVAL and f"of {backward} bytes" in refusal
        got[cus] = forward, backward
    assert got[32][0] < got[256][0] and got[32][1] < got[256][1], "fewer CUs, fewer shares"


def test_heads_of_a_kv_head(nxg):
    """A tile's reach over 128 tokens is counted in 32 bits: 128 * 65,536 heads * 16 pieces of a head are 2^27."""
    L = nxg.load_library()
    for f in (L.nxg_attention_rows_workspace_bytes, L.nxg_attention_rows_backward_workspace_bytes):
        assert f(ctypes.byref(params(nxg, n_head=1 << 16, n_kv_head=1))) >= 0
        assert f(ctypes.byref(params(nxg, n_head=(1 << 16) + 1, n_kv_head=1))) == -nxg.NXG_EINVAL
    refused(nxg, L, forward(nxg, L, params(nxg, n_head=1 << 20, n_kv_head=1, T_q=128)), "n_head=1048576")
