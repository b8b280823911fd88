"""The waits of attention's kernels of 128 rows, checked on the built code (no GPU needed).

Each wave loads its quarter of a step's codes and scales straight into a ring of four steps in
LDS, for all the waves of its workgroup, and passes a barrier once its own loads of the next step
have landed: loads return in the order they were issued, so after `s_waitcnt vmcnt(n)` all but the
last n have.  The compiler may put other loads among them (spilled registers, the scales of NaN
blocks), which only makes a wait longer; so what is checked is that between two barriers a wave
issues the loads of one step, and that the wait before a barrier leaves no more than those of two
in flight (three in the prologue)."""
from __future__ import annotations

import ctypes
import re
import shutil
import subprocess

import pytest

OBJDUMP = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"
DIMS = (64, 128, 192, 256)
TYPES = ("bf16", "f16", "f32")


@pytest.fixture(scope="module")
def kernels(axc, tmp_path_factory):
    """name -> instructions of every kernel of attention's code object."""
    if not shutil.which(OBJDUMP):
        pytest.skip("llvm-objdump is not installed")
    lib = axc.load_library()
    begin, end = (ctypes.addressof(ctypes.c_char.in_dll(lib, f"axh_kv_attention_co_{n}"))
                  for n in ("begin", "end"))
    co = tmp_path_factory.mktemp("co") / "kv_attention.co"
    co.write_bytes(ctypes.string_at(begin, end - begin))
    text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(co)], check=True, text=True,
                          stdout=subprocess.PIPE).stdout
    out: dict = {}
    for line in text.splitlines():
        if m := re.match(r"^[0-9a-f]+ <(\w+)>:", line):
            out[m.group(1)] = body = []
        elif line.startswith("\t"):
            body.append(line.split("//")[0].strip())
    return out


def _steps(body):
    """(loads into LDS since the barrier before, instruction before it, whether all loads were
    waited for behind the last of them) of each barrier, in address order: prologue, a step that
    is looked at and one that is not, what follows."""
    out, loads, drained = [], 0, False
    for before, ins in zip([""] + body, body):
        if ins.startswith("buffer_load") and ins.endswith("lds"):
            loads += 1
            drained = False
        elif ins.startswith("s_waitcnt") and "vmcnt(0)" in ins:
            drained = True
        elif ins.split()[0] == "s_barrier":
            out.append((loads, before, drained))
            loads = 0
    return out


def _in_order(body, step):
    at = _steps(body)
    loads = [n for n, _, _ in at]
    waits = [int(m[1]) if (m := re.search(r"vmcnt\((\d+)\) lgkmcnt\(0\)", w)) else None
             for _, w, _ in at[:4]]
    # four steps, then one at a barrier (two copies of the loop's body), then no more
    return (loads == [4 * step, 0, step, step] + [0] * (len(at) - 4) and len(at) > 4
            and waits == [3 * step, 2 * step, 2 * step, 2 * step]
            and at[4][2])  # all have landed before LDS is used for something else


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("dim", DIMS)
def test_steps_have_landed_at_their_barriers(kernels, dim, t):
    body = kernels[f"axh_kv_attention_many_d{dim}_{t}"]
    assert _in_order(body, 2 if dim <= 128 else 4), _steps(body)


def test_a_longer_wait_or_a_missing_load_would_be_seen(kernels):
    body = kernels["axh_kv_attention_many_d128_bf16"]
    assert not _in_order([i.replace("vmcnt(4) lgkmcnt(0)", "vmcnt(6) lgkmcnt(0)") for i in body], 2)
    assert not _in_order([i.replace("vmcnt(0)", "vmcnt(1)") for i in body], 2)
    last = max(i for i, x in enumerate(body) if x.startswith("buffer_load") and x.endswith("lds"))
    assert not _in_order(body[:last] + body[last + 1:], 2)


def test_few_rows_do_not_spill(kernels):
    for name, body in kernels.items():
        if "_many_" not in name:
            assert not any(i.startswith("scratch_") for i in body), name
