"""The serving operators on the CPU, lane by lane (test infrastructure).

`build()` compiles their translation units against lanes/hip/hip_runtime.h under
AddressSanitizer and UBSan, and links them with the rest of the CPU build (build.py)
and lanes_main.cpp; `Program` collects buffers and calls, runs them there and gives
the buffers back.
"""
from __future__ import annotations

import concurrent.futures as cf
import os
import subprocess
import sys
import tempfile

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, HERE)
import build as emu_build  # noqa: E402  (tests/cpu_emu/build.py)

EXE = os.path.join(emu_build.OUT_DIR, "emu_lanes")
UNITS = ["rmsnorm", "kv", "matvec_q4g", "paged_attention"]
HEADER = os.path.join(HERE, "lanes", "hip", "hip_runtime.h")


def _object(cpp: str, out: str, inputs: list[str]) -> str:
    if emu_build._stale(out, [*inputs, HEADER, os.path.abspath(__file__), *emu_build._deps()]):
        res = subprocess.run([emu_build.CLANG, "-I", os.path.join(HERE, "lanes"), *emu_build.FLAGS, "-O1", "-c", cpp, "-o", out],
                             capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"clang++ failed for {cpp}:\n{res.stderr[-6000:]}")
    return out


def build() -> str:
    emu_build.build()
    out = emu_build.OUT_DIR
    jobs = [(os.path.join(out, u + ".cpp"), os.path.join(out, u + "_lanes.o"), [os.path.join(out, u + ".cpp")]) for u in UNITS]
    main = os.path.join(HERE, "lanes_main.cpp")
    jobs.append((main, os.path.join(out, "lanes_main.o"), [main]))
    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        objs = list(ex.map(lambda j: _object(*j), jobs))
    rest = [os.path.splitext(s)[0] for s in emu_build.sources()]
    objs += [os.path.join(out, s + ".o") for s in rest if s not in UNITS]
    if emu_build._stale(EXE, objs):
        res = subprocess.run([emu_build.CLANG, "-fsanitize=address,undefined", *objs, "-o", EXE], capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"link failed:\n{res.stderr[-4000:]}")
    return EXE


class Fault(Exception):
    """A bad access, undefined behaviour, or a lane missing from a matrix instruction."""


class Program:
    """Buffers and calls, in the order in which they run.

    `cus`: compute units of the emulated GPU; `reverse`: blocks and waves from the last to the first."""

    def __init__(self, cus: int = 256, reverse: bool = False):
        self.lines, self.arrays, self.env = [], [], {"EMU_CUS": str(cus), "EMU_REVERSE": "1" if reverse else "0"}
        self.codes, self.allocations, self.messages = [], [], []

    def buf(self, array: np.ndarray, short: int = 0) -> int:
        """A device buffer with the array's bytes, the last `short` left out; its number."""
        raw = np.ascontiguousarray(array).reshape(-1).view(np.uint8)
        raw = raw[:len(raw) - short]
        self.arrays.append((raw, np.ascontiguousarray(array)))
        self.lines.append(f"buf {len(raw)}")
        return len(self.arrays) - 1

    def call(self, name: str, *args) -> None:
        """Arguments: numbers, None, ("b", buffer) or ("b", buffer, byte offset)."""
        def text(a):
            if a is None:
                return "null"
            if isinstance(a, tuple):
                return f"b{a[1]}+{a[2] if len(a) > 2 else 0}"
            return repr(a)

        self.lines.append(" ".join(["call", name, *map(text, args)]))

    def run(self, timeout: int = 600) -> list[np.ndarray]:
        """The buffers after the calls, shaped as they went in."""
        with tempfile.TemporaryDirectory() as d:
            program, data = os.path.join(d, "program"), os.path.join(d, "data")
            with open(program, "w") as f:
                f.write("\n".join(self.lines) + "\n")
            with open(data, "wb") as f:
                for raw, _ in self.arrays:
                    f.write(raw.tobytes())
            p = subprocess.run([EXE, program, data], capture_output=True, text=True, timeout=timeout,
                               env={**os.environ, **self.env, "ASAN_OPTIONS": "detect_leaks=0:detect_stack_use_after_return=0"})
            if p.returncode != 0:
                lines = [ln for ln in p.stderr.splitlines() if "ERROR" in ln or "runtime error" in ln or "    #" in ln]
                raise Fault("\n".join(lines[:12]) or f"exit {p.returncode}: {p.stderr[-2000:]}")
            for ln in p.stdout.splitlines():
                _, code, alive, *message = ln.split(" ", 3)
                self.codes.append(int(code))
                self.allocations.append(int(alive))
                self.messages.append(message[0] if message else "")
            with open(data, "rb") as f:
                raw = f.read()
        out, at = [], 0
        for r, a in self.arrays:
            got = np.frombuffer(raw[at:at + len(r)], dtype=np.uint8)
            at += len(r)
            out.append(got.view(a.dtype).reshape(a.shape).copy() if len(r) == a.nbytes else got.copy())
        return out
