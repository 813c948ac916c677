"""The products' kernels read fragments from LDS by asm, whose outputs are there only behind the wait after them; the compiler does
not know that.  So the built kernels are read: no instruction touches a register that an LDS read still in flight writes (a copy
or a spill of it would), on any path, and none of the kernels has scratch memory.  On the disassembly of libcx_moe.so."""
from __future__ import annotations

import os
import re
import subprocess
from pathlib import Path

import pytest

from constellation_amd.build import HIPCC, LIB

LLVM = Path(os.environ.get("CX_LLVM_BIN", Path(HIPCC).resolve().parent.parent / "lib" / "llvm" / "bin"))
if not LLVM.exists():
    LLVM = Path("/opt/rocm/llvm/bin")

KERNELS = ("k_mm", "k_mm_dx", "k_mm_dw", "k_mm_dw_short")  # those with fragments
REG = re.compile(r"\bv(?:\[(\d+):(\d+)\]|(\d+))")
WAIT = re.compile(r"lgkmcnt\((\d+)\)")
FAR = 16  # lgkmcnt counts no further


def registers(text):
    out = set()
    for lo, hi, one in REG.findall(text):
        out.update(range(int(lo), int(hi) + 1) if lo else (int(one),))
    return out


class Step:
    """What an instruction does to reads in flight."""
    __slots__ = ("wait", "touch", "fill", "counts", "text", "to", "falls")

    def __init__(self, text, to):
        op, _, args = text.partition(" ")
        self.text, self.to = text, to
        self.wait = int(WAIT.search(text).group(1)) if op == "s_waitcnt" and "lgkmcnt" in text else None
        self.counts = op.startswith(("ds_", "s_load", "s_store", "s_buffer_load", "flat_"))
        self.falls = op not in ("s_branch", "s_endpgm", "s_setpc_b64")
        self.touch, self.fill = registers(args), set()
        if op.startswith("ds_read"):
            first, _, rest = args.partition(",")
            self.fill, self.touch = registers(first), registers(rest)  # reads land in order: one may follow another into a register


def faults(steps):
    """Instructions that touch a register of a read in flight, on some path.  A state is {register: LDS operations issued since}."""
    at, labels = {0: {}}, {s.to for s in steps}
    work, bad = [0], {}
    while work:
        i = work.pop()
        held = dict(at[i])
        while True:
            s = steps[i]
            if s.wait is not None:
                held = {r: n for r, n in held.items() if n < s.wait}
            hit = s.touch & held.keys()
            if hit:
                bad[i] = s.text
                for r in hit:
                    del held[r]
            if s.counts:
                held = {r: n + 1 for r, n in held.items() if n + 1 < FAR}
                held.update((r, 0) for r in s.fill)
            nexts = ([i + 1] if s.falls else []) + ([s.to] if s.to is not None else [])
            if len(nexts) == 1 and nexts[0] == i + 1 and i + 1 not in labels:
                i += 1
                continue
            for n in nexts:
                known = at.get(n)
                merged = dict(held) if known is None else {r: min(held.get(r, FAR), known.get(r, FAR)) for r in held.keys() | known.keys()}
                if merged != known:
                    at[n] = merged
                    work.append(n)
            break
    return bad


def kernels(path):
    """(name, steps) of each kernel in a code object's disassembly."""
    text = subprocess.run([LLVM / "llvm-objdump", "-d", "--no-show-raw-insn", str(path)], capture_output=True, text=True, check=True).stdout
    name, lines = None, []
    for line in [*text.splitlines(), "0 <end>:"]:
        head = re.match(r"([0-9a-f]+) <(.+)>:$", line)
        if head:
            if name:
                yield name, lines
            name, start, lines = head.group(2), int(head.group(1), 16), []
            continue
        m = re.match(r"\t(.*?)\s*// ([0-9A-F]+):(.*)", line)
        if not m:
            continue
        to = re.search(r"<[^>+]+(?:\+0x([0-9a-f]+))?>", m.group(3)) if m.group(1).startswith(("s_branch", "s_cbranch")) else None
        lines.append((int(m.group(2), 16), m.group(1), None if to is None else start + int(to.group(1) or "0", 16)))


def steps_of(lines):
    index = {a: i for i, (a, _, _) in enumerate(lines)}
    return [Step(text, None if t is None else index[t]) for _, text, t in lines]


@pytest.fixture(scope="module")
def objects(tmp_path_factory):
    if not LIB.exists() or not (LLVM / "llvm-objdump").exists():
        pytest.skip("no built library or no disassembler")
    d = tmp_path_factory.mktemp("objects")
    (d / "lib.so").symlink_to(LIB)
    subprocess.run([LLVM / "llvm-objdump", "--offloading", "lib.so"], cwd=d, check=True, capture_output=True)
    return [f for f in sorted(d.iterdir()) if "gfx950" in f.name and b"k_mm" in f.read_bytes()]


def of_the_products(name):
    m = re.search(r"(\d+)(k_mm\w*?)I", name)
    return m is not None and m.group(2)[:int(m.group(1))] in KERNELS


def test_the_check_finds_what_it_looks_for():
    """An early use, an early overwrite, a use on one of two paths, and a wait that leaves one read in flight."""
    def bad(*text, to={}):
        return sorted(faults([Step(t, to.get(i)) for i, t in enumerate(text)]))
    read = "ds_read_b128 v[4:7], v0 offset:16"
    assert bad(read, "s_waitcnt lgkmcnt(0)", "v_mfma v[8:11], v[4:7], v[4:7], 0", "s_endpgm") == []
    assert bad(read, "v_mov_b32_e32 v9, v5", "s_endpgm") == [1]
    assert bad(read, "v_mov_b32_e32 v5, 0", "s_endpgm") == [1]
    assert bad(read, "scratch_store_dwordx4 off, v[4:7], off", "s_endpgm") == [1]
    assert bad(read, "ds_read_b128 v[8:11], v0", "s_waitcnt lgkmcnt(1)", "v_mov_b32_e32 v0, v4", "v_mov_b32_e32 v0, v8", "s_endpgm") == [4]
    assert bad(read, "s_cbranch_scc1 2", "s_waitcnt vmcnt(0) lgkmcnt(0)", "v_mov_b32_e32 v0, v4", "s_endpgm", to={1: 3}) == [3]
    assert bad("s_waitcnt lgkmcnt(0)", "v_mov_b32_e32 v0, v4", read, "s_cbranch_scc1 0", "s_endpgm", to={3: 0}) == []
    assert bad("v_mov_b32_e32 v0, v4", read, "s_cbranch_scc1 0", "s_endpgm", to={2: 0}) == [0]


def test_no_read_in_flight_is_touched(objects):
    seen, reads = 0, 0
    for path in objects:
        for name, lines in kernels(path):
            if not of_the_products(name):
                continue
            steps = steps_of(lines)
            seen, reads = seen + 1, reads + sum(bool(s.fill) for s in steps)
            bad = faults(steps)
            assert not bad, (name, list(bad.items())[:4])
    assert seen >= 22 and reads > 5000, (seen, reads)


def test_no_scratch_memory(objects):
    seen = 0
    for path in objects:
        notes = subprocess.run([LLVM / "llvm-readelf", "--notes", str(path)], capture_output=True, text=True, check=True).stdout
        for entry in notes.split("- .agpr_count")[1:]:
            name = re.search(r"\.name:\s+(\S+)", entry).group(1)
            if of_the_products(name):
                seen += 1
                assert re.search(r"\.private_segment_fixed_size:\s+0\b", entry) and re.search(r"\.vgpr_spill_count:\s+0\b", entry), name
    assert seen >= 22, seen
