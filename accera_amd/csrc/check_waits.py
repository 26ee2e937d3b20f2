"""Looks through the device code of a built library for instructions that come too soon behind one whose result they read.

The gfx9 instruction set leaves some waits to the program (its tables of wait states that software has to insert).  The compiler keeps them between the
instructions that it knows, but it does not look into inline assembly: what stands there has to hold for whatever the register allocator puts in front of it, a scalar
register brought back from its spill slot with v_readlane included.  Whether it does is a matter of each build, so the built code is what is read:

  a vector instruction writes a scalar register (or vcc), a memory instruction reads it        5 instructions between
  ...                                                     a vector instruction reads it        2
  ...                                                     v_readlane / v_writelane by its lane 4
  a vector instruction writes a vector register, v_readlane / v_readfirstlane reads it         1
  ...                                            a DPP operand                                 2
  a transcendental instruction's result, another vector instruction reads it                   1

(Matrix instructions, whose waits depend on their shapes, are the compiler's here or have a check of their own.)  Code is read in the order it lies in.

    python3 check_waits.py <library .so> [...]
"""
import concurrent.futures
import re
import struct
import subprocess
import sys
import tempfile

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
_BUNDLE = b"__CLANG_OFFLOAD_BUNDLE__"

_MEMORY = re.compile(r"(global|buffer|flat|scratch|tbuffer)_")
_TRANSCENDENTAL = re.compile(r"v_(exp|log|rcp|rsq|sqrt|sin|cos)_(f16|f32|f64|iflag)")
_NO_SCALAR_RESULT = re.compile(r"s_(cmp|bitcmp|waitcnt|barrier|nop|cbranch|branch|endpgm|set)")
_TWO_RESULTS = re.compile(r"_co_|div_scale|mad_[iu]64|swap")
_READS_RESULT = re.compile(r"v_(fmac|mac|fmamk|writelane|dot\w*c_)|swap")


def code_objects(path):
    """The gfx950 code objects inside a library, one for each translation unit."""
    data = open(path, "rb").read()
    at = data.find(_BUNDLE)
    while at >= 0:
        entry = at + len(_BUNDLE) + 8
        for _ in range(struct.unpack_from("<Q", data, entry - 8)[0]):
            offset, size, text = struct.unpack_from("<QQQ", data, entry)
            if b"gfx950" in data[entry + 24:entry + 24 + text] and size:
                yield data[at + offset:at + offset + size]
            entry += 24 + text
        at = data.find(_BUNDLE, at + 1)


def _registers(text, kinds="sv"):
    out = set()
    for kind, first, last, one in re.findall(r"(?<![\w.])([%s])(?:\[(\d+):(\d+)\]|(\d+))(?!\w)" % kinds, text):
        out |= {kind + str(i) for i in (range(int(first), int(last) + 1) if first else (int(one),))}
    if "s" in kinds and re.search(r"(?<!\w)vcc(?!\w)", text):
        out.add("svcc")
    return out


def _waits(op, args):
    """(what it is, instructions between, registers, only behind transcendental ones) for what an instruction reads."""
    if _MEMORY.match(op):
        return [("vector write of a scalar register, memory read", 5, _registers(", ".join(args), "s"), False)]
    if not op.startswith("v_") or op.startswith(("v_mfma", "v_smfma")):
        return []
    results = 2 if _TWO_RESULTS.search(op) else 1
    reads = _registers(", ".join(args if _READS_RESULT.search(op) else args[results:]))
    out = [("vector write of a scalar register, vector read", 2, {r for r in reads if r[0] == "s"}, False)]
    if not _TRANSCENDENTAL.match(op):
        out.append(("transcendental result, vector read", 1, {r for r in reads if r[0] == "v"}, True))
    if op.startswith(("v_readlane", "v_readfirstlane")):
        out.append(("vector write of a vector register, read of a lane", 1, _registers(args[1], "v"), False))
    if op.startswith(("v_readlane", "v_writelane")):
        out.append(("vector write of a scalar register, number of a lane", 4, _registers(args[-1], "s"), False))
    if "_dpp" in op:
        out.append(("vector write of a vector register, DPP read", 2, _registers(args[1].split()[0], "v"), False))
    return out


def violations(lines):
    """(kernel, what, writer, reader) of each instruction in a disassembly that comes too soon."""
    kernel, recent = None, []  # (instruction, registers a vector instruction wrote, further waits, transcendental), oldest first
    for line in lines:
        m = re.match(r"[0-9a-f]+ <(.*)>:", line)
        if m:
            kernel, recent = m.group(1), []
            continue
        line = line.split("//")[0].strip()
        m = re.match(r"([a-z]+_\w+)(?:\s+(.*))?$", line)
        if not m:
            continue
        op, args = m.group(1), [a.strip() for a in (m.group(2) or "").split(",")]
        for what, between, registers, transcendental in _waits(op, args):
            passed = 0
            for writer, wrote, more, fast in reversed(recent):
                if passed >= between:
                    break
                if wrote & registers and (fast or not transcendental):
                    yield kernel, what, writer, line
                passed += 1 + more
        wrote = set()
        if op.startswith("v_") and not op.startswith(("v_mfma", "v_smfma", "v_nop")):
            wrote = _registers(", ".join(args[:2 if _TWO_RESULTS.search(op) else 1]))
        elif op.startswith("s_") and not _NO_SCALAR_RESULT.match(op):
            over = _registers(args[0], "s")  # (what a scalar instruction writes is waited for)
            recent = [(w, r - over, n, t) for w, r, n, t in recent]
        recent.append((line, wrote, int(args[0]) if op == "s_nop" else 0, bool(_TRANSCENDENTAL.match(op))))
        del recent[:-8]


def _of_code(blob):
    with tempfile.NamedTemporaryFile(suffix=".co") as f:
        f.write(blob)
        f.flush()
        p = subprocess.Popen([OBJDUMP, "-d", "--no-show-raw-insn", "--mcpu=gfx950", f.name], stdout=subprocess.PIPE, text=True)
        found = list(violations(p.stdout))
        if p.wait():
            raise RuntimeError(f"{OBJDUMP} ended with {p.returncode}")
    return found


def check(paths, workers=8):
    """(code objects read, violations)"""
    blobs = sorted((b for path in paths for b in code_objects(path)), key=len, reverse=True)
    with concurrent.futures.ProcessPoolExecutor(workers) as pool:
        return len(blobs), [v for found in pool.map(_of_code, blobs) for v in found]


def main(paths):
    read, found = check(paths)
    for kernel, what, writer, reader in found[:40]:
        print(f"{kernel}: {what}: {writer} ... {reader}", file=sys.stderr)
    if not read:
        print("no gfx950 code found in " + ", ".join(paths), file=sys.stderr)
    return 1 if found or not read else 0


if __name__ == "__main__":
    sys.exit(main(sys.argv[1:]))
