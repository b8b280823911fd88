"""The waits of the MXFP4 tile kernels, checked on the built code (no GPU needed).

Every wave loads codes into LDS for all the waves of its workgroup and passes a
barrier once its own loads of the next step have landed, which it tells from the
load counter: loads return in the order they were issued, so after `s_waitcnt
vmcnt(n)` all but the last n have.  n also leaves room for loads of scales, whose
place among the others the compiler chooses: so it is checked on the instructions
that at no barrier more loads into LDS are in flight than those of the steps
behind the next one."""
from __future__ import annotations

import ctypes
import re
import shutil
import subprocess

import pytest

OBJDUMP = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"
# tile -> loads of a wave and step, buffers
TILES = {"t64x64": (8, 3), "t64x128": (6, 3), "t128x128": (8, 2), "t256x256": (8, 2)}


@pytest.fixture(scope="module")
def kernels(axc, tmp_path_factory):
    """name -> instructions of every kernel of the MXFP4 matmul code object."""
    if not shutil.which(OBJDUMP):
        pytest.skip("llvm-objdump is not installed")
    lib = axc.load_library()
    begin, end = (ctypes.addressof(ctypes.c_char.in_dll(lib, f"axh_mx_matmul_co_{n}"))
                  for n in ("begin", "end"))
    co = tmp_path_factory.mktemp("co") / "mx_matmul.co"
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


def _in_flight(body, extra=None):
    """Loads into LDS in flight at every barrier, along the instructions in address
    order (prologue, one turn of the loop, what follows: a branch back enters where
    the fall-through does).  `extra`: added to every wait, a planted mistake."""
    loads, out = [], []
    for ins in body:
        op = ins.split()[0]
        if op.startswith(("buffer_load", "global_load")):
            loads.append(ins.endswith("lds"))
        elif op == "s_waitcnt":
            if m := re.search(r"vmcnt\((\d+)\)", ins):
                n = int(m.group(1)) + (extra or 0)
                loads = loads[len(loads) - n:] if n and n < len(loads) else loads if n else []
        elif op == "s_barrier":
            out.append(sum(loads))
    return out


@pytest.mark.parametrize("tile", TILES)
def test_the_next_step_has_landed_at_every_barrier(kernels, tile):
    per_step, buffers = TILES[tile]
    named = [n for n in kernels if f"_{tile}_" in n]
    assert len(named) == 10  # matmul, expert matmul: 3 types; gate/up: 4
    for name in named:
        at = _in_flight(kernels[name])
        assert len(at) >= 4, name  # prologue, two steps, the end
        # step 0 alone in the prologue: half of the last buffer's loads come in the loop
        assert at[0] <= (buffers - 2) * per_step + per_step // 2, name
        assert max(at[1:]) <= (buffers - 2) * per_step, name
        assert at[-1] == 0, name  # before LDS is used for the results


@pytest.mark.parametrize("tile", TILES)
def test_a_longer_wait_would_be_seen(kernels, tile):
    per_step, buffers = TILES[tile]
    body = kernels[f"axh_mxfp4_matmul_{tile}_f32"]
    assert max(_in_flight(body, extra=2)[1:]) > (buffers - 2) * per_step


def test_no_kernel_spills(kernels):
    for name, body in kernels.items():
        assert not any(i.startswith("scratch_") for i in body), name
