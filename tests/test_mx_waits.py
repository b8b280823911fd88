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
# tile -> loads of a wave and step, of them of A, and buffers
TILES = {"t64x64": (8, 4, 3), "t64x64s2": (8, 4, 3), "t64x128": (6, 2, 3), "t128x64": (6, 4, 3),
         "t128x128": (8, 4, 2), "t128x128n": (8, 4, 2), "t256x256": (8, 4, 2)}


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


def _named(kernels, tile):
    named = [n for n in kernels if f"_{tile}_" in n]
    # dense products: 3 types; expert layers: 3, gate/up: 4
    assert len(named) == {"t64x64": 3, "t64x64s2": 3, "t64x128": 3, "t128x64": 7}.get(tile, 10)
    return named


@pytest.mark.parametrize("tile", TILES)
def test_the_next_step_has_landed_at_every_barrier(kernels, tile):
    per_step, _, buffers = TILES[tile]
    for name in _named(kernels, tile):
        at = _in_flight(kernels[name])
        assert len(at) >= 4, name  # prologue, two steps, the end
        # step 0 alone in the prologue: half of the last buffer's loads come in the loop
        assert at[0] <= (buffers - 2) * per_step + per_step // 2, name
        assert max(at[1:]) <= (buffers - 2) * per_step, name
        assert at[-1] == 0, name  # before LDS is used for the results


def _descriptors(body):
    """The buffer descriptor of each load into LDS, and None for each barrier."""
    out = []
    for ins in body:
        if ins.split()[0] == "s_barrier":
            out.append(None)
        elif ins.endswith("lds") and ins.startswith("buffer_load"):
            out.append(re.search(r"s\[\d+:\d+\]", ins)[0])
    return out


@pytest.mark.parametrize("tile", TILES)
def test_loads_come_in_the_order_that_the_waits_count_on(kernels, tile):
    """A and X of all buffers but the last, then the last buffer's first half; in the
    loop, second half, barrier, first half.  (With the last buffer's before X of the
    others, the count at a barrier is the same, but the younger loads are not.)"""
    per_step, of_a, buffers = TILES[tile]
    step = [False] * of_a + [True] * (per_step - of_a)
    half = per_step // 2
    want = ([False] * of_a * (buffers - 1) + [True] * (per_step - of_a) * (buffers - 1)
            + step[:half] + [None] + (step[half:] + [None] + step[:half]) * 2 + [None])
    for name in _named(kernels, tile):
        loads = _descriptors(kernels[name])
        x = loads[of_a * (buffers - 1)]  # the first that has to be X's
        assert [v if v is None else v == x for v in loads[:len(want)]] == want, name


@pytest.mark.parametrize("tile", TILES)
def test_a_longer_wait_would_be_seen(kernels, tile):
    per_step, _, buffers = TILES[tile]
    body = kernels[_named(kernels, tile)[0]]
    assert max(_in_flight(body, extra=2)[1:]) > (buffers - 2) * per_step


def test_no_kernel_spills(kernels):
    for name, body in kernels.items():
        assert not any(i.startswith("scratch_") for i in body), name
