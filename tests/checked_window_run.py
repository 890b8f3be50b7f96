"""Runs the checked build (libodf_sm100_checked.so) over sliding-window problems and prints one JSON line per
case: the status word and the failed in-kernel invariants.  Started as its own process by
tests/test_window_gpu.py, so that the checked library is the only copy of the library in it.
"""
from __future__ import annotations

import ctypes as C
import json
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent
sys.path.insert(0, str(ROOT / "dnn-flash_b200"))

import odf_b200  # noqa: E402

odf_b200.LIB_PATH = ROOT / "dnn-flash_b200" / "lib" / "libodf_sm100_checked.so"

import torch  # noqa: E402


def main():
    for case in (dict(D=128, M=1500, N=1500, window=384, sinks=4), dict(D=64, M=700, N=700, window=100, sinks=200),
                 dict(D=128, M=200, N=9000, window=7000, sinks=130), dict(D=128, M=900, N=900, window=128, alibi=True),
                 dict(D=64, M=600, N=400, window=50, softcap=20.0), dict(D=128, M=300, N=300, window=1, sinks=1)):
        D, M, N = case.pop("D"), case.pop("M"), case.pop("N")
        q, k, v = (torch.randn((2, h, t, D), device="cuda").to(torch.bfloat16) for h, t in ((4, M), (2, N), (2, N)))
        off = max(0, N - M)
        odf_b200.flash_fwd_window(q, k, v, q_offset=off, **case)
        torch.cuda.synchronize()
        bits = C.c_uint32(0)
        rc = odf_b200.load_library().odf_debug_check_bits(C.byref(bits))
        print(json.dumps({"case": [D, M, N, case], "rc": rc, "check_bits": bits.value, "status": odf_b200.device_status()}),
              flush=True)


if __name__ == "__main__":
    main()
