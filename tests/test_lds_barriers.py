"""No wave of any kernel of the built library reaches a barrier with LDS writes of its own under way: what the others read
behind the barrier has been written.  The compiler sees to it for __syncthreads, but not everywhere: it has left the
wait out where a loop ends with a write and begins with the barrier.  So the library's own device code is read back:
a wave's operations on LDS end in order, and s_waitcnt lgkmcnt(n) leaves the last n of them."""
import glob
import os
import re
import shutil
import subprocess

import pytest

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
NONE = 99  # no write under way
WRITE = re.compile(r"ds_(write|add|sub|max|min|or|and|xor|inc|dec|cmpst|wrxchg)")


def kernels(listing):
    """(name, [(address, operation, arguments, branch target or None)]) of a disassembly."""
    name, body = None, []
    for line in listing.splitlines():
        m = re.match(r"^(?:[0-9a-f]+ )?<(\w+)>:$", line)
        if m:
            if body:
                yield name, body
            name, body = m.group(1), []
            continue
        m = re.match(r"^\s+(\S+)\s*(.*?)\s*// ([0-9A-F]+):[^<]*(?:<\w+?(?:\+0x([0-9a-f]+))?>)?$", line)
        if m and name:
            op, args, at, off = m.groups()
            at = int(at, 16)
            start = body[0][0] if body else at
            body.append((at, op, args, start + int(off or "0", 16) if op.startswith(("s_cbranch", "s_branch")) else None))
    if body:
        yield name, body


def open_writes(body):
    """Addresses of the barriers that may be reached with a write under way: how many operations ago the last one was, over
    all paths."""
    place = {ins[0]: i for i, ins in enumerate(body)}
    state, work, found = {0: NONE}, [0], set()
    while work:
        i = work.pop()
        ago, (at, op, args, target) = state[i], body[i]
        if WRITE.match(op):
            ago = 1
        elif op.startswith(("ds_", "s_load", "s_buffer_load", "s_memtime")):
            ago = min(NONE, ago + 1)
        elif op == "s_waitcnt":
            m = re.search(r"lgkmcnt\((\d+)\)", args)
            if args == "0" or (m and int(m.group(1)) < ago):
                ago = NONE
        elif op == "s_barrier" and ago < NONE:
            found.add(at)
        following = [] if op in ("s_branch", "s_endpgm") else [i + 1]
        if target is not None:
            following.append(place[target])
        for j in following:
            if j < len(body) and ago < state.get(j, NONE + 1):
                state[j] = ago
                work.append(j)
    return found


LOOP = """
<loop>:
	s_mov_b32 s0, 0                                            // 000000000100: BE800080
	{wait}                                                     // 000000000104: BF8C0F70
	s_barrier                                                  // 000000000108: BF8A0000
	ds_read_b32 v1, v0                                         // 00000000010C: D86C0000 01000000
	s_waitcnt lgkmcnt(0)                                       // 000000000114: BF8CC07F
	ds_write_b32 v0, v1                                        // 000000000118: D81A0000 00000100
	ds_read_b32 v2, v0 offset:4                                // 000000000120: D86C0004 02000000
	s_cbranch_scc1 65526                                       // 000000000128: BF85FFF6 <loop+0x4>
	s_endpgm                                                   // 00000000012C: BF810000
"""


@pytest.mark.parametrize("wait,found", [("s_waitcnt vmcnt(0)", {0x108}), ("s_waitcnt vmcnt(0) lgkmcnt(0)", set()),
                                        ("s_waitcnt lgkmcnt(1)", set()), ("s_waitcnt lgkmcnt(2)", {0x108}), ("s_waitcnt 0", set())])
def test_the_search_finds_a_missing_wait(wait, found):
    (name, body), = kernels(LOOP.format(wait=wait))
    assert name == "loop" and len(body) == 9 and open_writes(body) == found


def test_no_writes_open_at_a_barrier(ie, tmp_path):
    lib = str(tmp_path / "lib.so")
    shutil.copy(ie.LIB_PATH, lib)
    subprocess.run([OBJDUMP, "--offloading", lib], cwd=tmp_path, check=True, capture_output=True)
    count, bad = 0, []
    for part in sorted(glob.glob(lib + ".*gfx950")):
        text = subprocess.run([OBJDUMP, "-d", part], check=True, capture_output=True, text=True).stdout
        for name, body in kernels(text):
            count += sum(op == "s_barrier" for _, op, _, _ in body)
            bad += [(name, hex(at)) for at in sorted(open_writes(body))]
    assert count > 1000 and os.path.getsize(lib) > 0
    assert not bad, f"{len(bad)}: {bad[:5]}"
