"""Which kernel flash_decode runs a call as (csrc/decode_plan.h, compiled for the host), for the tests."""
import collections
import ctypes
import functools
import os
import subprocess
import tempfile

from conftest import ROOT

Plan = collections.namedtuple("Plan", "wide part_rows row_tiles items cluster ctas tiles")


@functools.cache
def _library():
    folder = tempfile.mkdtemp()
    so = os.path.join(folder, "decode_plan.so")
    csrc = os.path.join(ROOT, "flash-attn-rtx5060_b200", "csrc")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", csrc, "-o", so,
                           os.path.join(ROOT, "tests", "decode_plan_host.cpp")])
    return ctypes.CDLL(so)


def plan(batch, tokens, q_heads, kv_heads, room, head_dim, window_left=-1):
    out = (ctypes.c_longlong * 7)()
    _library().plan((ctypes.c_longlong * 7)(batch, tokens, q_heads // kv_heads, kv_heads, room, window_left, head_dim), out)
    return Plan(*out)
