"""The waits of the MXFP4 kernels whose waves load LDS for themselves, checked on the built
code (no GPU needed): the K-split products (a ring of buffers a wave) and the single-token
products (a unit's activations).

Loads return in the order they were issued, so after `s_waitcnt vmcnt(n)` all but the last n
have landed.  The compiler chooses the place of the scales' loads among those of the codes,
which the counts have to bear; so every way through a kernel is followed, with the loads in
flight, to the reads of LDS."""
from __future__ import annotations

import ctypes
import re
import shutil
import subprocess

import pytest

OBJDUMP = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"


def _code(axc, tmp_path_factory, name):
    """kernel -> its instructions as (address, text)."""
    if not shutil.which(OBJDUMP):
        pytest.skip("llvm-objdump is not installed")
    lib = axc.load_library()
    begin, end = (ctypes.addressof(ctypes.c_char.in_dll(lib, f"axh_{name}_co_{n}"))
                  for n in ("begin", "end"))
    co = tmp_path_factory.mktemp("co") / f"{name}.co"
    co.write_bytes(ctypes.string_at(begin, end - begin))
    text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(co)], check=True, text=True,
                          stdout=subprocess.PIPE).stdout
    out: dict = {}
    for line in text.splitlines():
        if m := re.match(r"^[0-9a-f]+ <(\w+)>:", line):
            out[m.group(1)] = body = []
        elif line.startswith("\t"):
            ins, _, at = line.partition("//")
            body.append((int(at.split(":")[0], 16), ins.strip()))
    return out


@pytest.fixture(scope="module")
def matmul(axc, tmp_path_factory):
    return _code(axc, tmp_path_factory, "mx_matmul")


@pytest.fixture(scope="module")
def matvec(axc, tmp_path_factory):
    return _code(axc, tmp_path_factory, "mx_matvec")


def _into_lds(ins):
    return ins.startswith("buffer_load") and ins.endswith("lds")


def _successors(body, places, i):
    at, ins = body[i]
    if not ins.startswith(("s_branch", "s_cbranch")):
        return [i + 1]
    words = int(ins.split()[1])
    to = places[at + 4 + 4 * (words - 65536 if words >= 32768 else words)]
    return [to] if ins.startswith("s_branch") else [i + 1, to]


def _left(queue, ins, extra):
    """The loads in flight after a wait; `extra`: added to its count, a planted mistake."""
    m = re.search(r"vmcnt\((\d+)\)", ins)
    n = int(m.group(1)) + extra if m else len(queue)
    return queue[max(0, len(queue) - n):] if n else ()


def _ring_holds(body, per_step, buffers, extra=0, turns=3):
    """Whether a step's codes have landed before its fragments are read, on every way from
    the first requests of the ring through `turns` turns of it."""
    places = {at: i for i, (at, _) in enumerate(body)}
    run = []  # the first `buffers` steps' requests: nothing is read or branched between them
    for i, (_, ins) in enumerate(body):
        if _into_lds(ins):
            run.append(i)
            if len(run) == buffers * per_step:
                break
        elif ins.startswith(("ds_read", "s_barrier", "s_branch", "s_cbranch")):
            run = []
    assert len(run) == buffers * per_step
    start = run[0]
    while not body[start - 1][1].startswith(("s_branch", "s_cbranch")):
        start -= 1
    todo, seen, done = [(start, (), 0, 0, False)], set(), 0
    while todo:
        state = todo.pop()
        if state in seen:
            continue
        seen.add(state)
        i, queue, asked, step, read = state
        ins = body[i][1]
        if ins.startswith(("buffer_", "global_")):
            lds = _into_lds(ins)
            queue += (asked if lds else -1,)
            asked += lds
            if read and asked == (buffers + step + 1) * per_step:
                step, read = step + 1, False
        elif ins.startswith("s_waitcnt"):
            queue = _left(queue, ins, extra)
        elif ins.startswith("ds_read"):
            if any(0 <= q < (step + 1) * per_step for q in queue):
                return False
            read = True
        elif ins.startswith("s_barrier"):  # past the ring
            continue
        done = max(done, step)
        if step < turns * buffers:
            todo += [(t, queue, asked, step, read) for t in _successors(body, places, i)]
    assert done == turns * buffers
    return True


# kernel -> loads of a step into LDS, buffers of a wave
RINGS = {"matmul_k16": (6, 3), "matmul_k32": (8, 2), "expert_matmul_k32": (8, 2),
         "expert_gate_up_k32": (12, 3)}


@pytest.mark.parametrize("kernel", RINGS)
def test_a_step_of_a_ring_has_landed_before_it_is_read(matmul, kernel):
    named = [n for n in matmul if n.startswith(f"axh_mxfp4_{kernel}_")]
    assert len(named) == (4 if "gate_up" in kernel else 3)
    for name in named:
        assert _ring_holds(matmul[name], *RINGS[kernel]), name


@pytest.mark.parametrize("kernel", RINGS)
def test_a_ring_with_longer_waits_would_be_seen(matmul, kernel):
    assert not _ring_holds(matmul[f"axh_mxfp4_{kernel}_f32"], *RINGS[kernel], extra=1)


def _stage_holds(body, extra=0):
    """Whether no load into LDS is in flight at any read of LDS, on every way through."""
    places = {at: i for i, (at, _) in enumerate(body)}
    todo, seen = [(0, ())], set()
    while todo:
        state = todo.pop()
        if state in seen:
            continue
        seen.add(state)
        i, queue = state
        ins = body[i][1]
        if ins.startswith("s_endpgm"):
            continue
        if ins.startswith(("buffer_", "global_")):
            queue += (_into_lds(ins),)
        elif ins.startswith("s_waitcnt"):
            queue = _left(queue, ins, extra)
        elif ins.startswith("ds_read") and any(queue):
            return False
        while queue and not queue[0]:  # no wait can leave what it does not hold up
            queue = queue[1:]
        todo += [(t, queue) for t in _successors(body, places, i)]
    return True


@pytest.mark.parametrize("lanes", [16, 32, 64])
@pytest.mark.parametrize("kernel", ["matvec", "expert_gate_up", "expert_down"])
def test_the_activations_have_landed_before_they_are_read(matvec, kernel, lanes):
    body = matvec[f"axh_mxfp4_{kernel}_l{lanes}"]
    assert sum(_into_lds(ins) for _, ins in body) == lanes // 8
    assert _stage_holds(body)
    assert not _stage_holds(body, extra=1)
