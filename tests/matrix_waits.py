"""Looks through gfx950 code for results of the matrix unit that are read before they are there.

A matrix instruction writes its result some cycles after it is issued, and only a following matrix instruction that adds to the same
registers waits by itself.  Anything else that reads them, or writes them, has to come a number of wait states later: 2 more than the
passes of an fp32 product, 4 more than those of a 16-bit one; every instruction is one state, s_nop n is n + 1.  The compiler puts the
waits in; where it does not (a product that ends a loop whose exit reads the sum at once), results are wrong without an error.
"""
import re
import struct
import subprocess

PASSES = {"4x4x4_16b_f32": (2, 2), "16x16x4_f32": (8, 2), "32x32x2_f32": (16, 2), "16x16x16_f16": (4, 4), "16x16x16_bf16": (4, 4),
          "16x16x32_f16": (4, 4), "16x16x32_bf16": (4, 4), "32x32x8_f16": (8, 4), "32x32x8_bf16": (8, 4), "32x32x16_f16": (8, 4),
          "32x32x16_bf16": (8, 4)}
_REG = re.compile(r"\b([va])(?:\[(\d+):(\d+)\]|(\d+)\b)")
_LINE = re.compile(r"^\s*(\S+)\s*(.*?)\s*//\s*([0-9A-Fa-f]+):((?:\s+[0-9A-Fa-f]{8})+)(?:\s*<.*>)?\s*$")


def code_objects(path):
    """The gfx950 code objects in a library built by hipcc."""
    data, at = open(path, "rb").read(), 0
    while True:
        at = data.find(b"__CLANG_OFFLOAD_BUNDLE__", at)
        if at < 0:
            return
        count, = struct.unpack_from("<Q", data, at + 24)
        p = at + 32
        for _ in range(count):
            off, size, n = struct.unpack_from("<QQQ", data, p)
            if b"gfx950" in data[p + 24:p + 24 + n]:
                yield data[at + off:at + off + size]
            p += 24 + n
        at += 24


def functions(objdump, path):
    """(name, [(operation, operands, index of a branch's target or None)]) of every function of a code object."""
    text = subprocess.run([objdump, "-d", path], check=True, capture_output=True, text=True).stdout
    for block in re.split(r"\n(?=[0-9a-f]{16} <)", text)[1:]:
        head, _, body = block.partition("\n")
        yield head.split("<", 1)[1].rstrip(">:"), parse(body)


def parse(body):
    ins, place = [], {}
    for line in body.splitlines():
        m = _LINE.match(line)
        if m:
            addr, words = int(m.group(3), 16), m.group(4).split()
            place[addr] = len(ins)
            ins.append((m.group(1), m.group(2), addr, len(words)))
    out = []
    for op, args, addr, _ in ins:
        target = None
        if op == "s_branch" or op.startswith("s_cbranch"):
            rel = int(args.split()[0], 0)
            target = place.get(addr + 4 + 4 * (rel - 65536 if rel >= 32768 else rel))
        out.append((op, args, target))
    return out


def registers(text):
    out = set()
    for kind, first, last, one in _REG.findall(text):
        out.update((kind, r) for r in (range(int(first), int(last) + 1) if first else (int(one),)))
    return out


def early(ins, writes=True):
    """(instruction, matrix instruction, its distance, the distance it needs) of every read of a result that comes too early, and of
    every write over one."""
    regs = {}

    def of(i):
        if i not in regs:
            op, args, _ = ins[i]
            parts = re.split(r",\s*(?![^\[]*\])", args)
            regs[i] = (registers(parts[0]), registers(",".join(parts[1:]))) if op.startswith("v_") else (set(), registers(args))
        return regs[i]

    for i, (op, args, _) in enumerate(ins):
        if not op.startswith("v_mfma"):
            continue
        shape = op[len("v_mfma_f32_"):]
        passes, more = PASSES[shape]
        need, result = passes + more, of(i)[0]
        seen, todo = {}, [(i + 1, 0)]
        while todo:
            j, gone = todo.pop()
            if j >= len(ins) or gone >= need or seen.get(j, need) <= gone:
                continue
            seen[j] = gone
            o, a, target = ins[j]
            if o == "s_endpgm":
                continue
            if o.startswith("v_mfma"):
                parts = re.split(r",\s*(?![^\[]*\])", a)
                if (registers(parts[1]) | registers(parts[2])) & result:
                    yield "%s %s" % (o, a), "%s %s" % (op, args), gone, need
                    continue
                if (of(j)[0] | registers(parts[3])) & result:
                    continue                                     # adds to the result, or replaces it: waits by itself
            elif o.startswith(("v_", "ds_", "global_", "buffer_", "flat_", "scratch_")):
                wrote, read = of(j)
                if wrote & result and not read & result and not writes:
                    continue
                if (wrote | read) & result:
                    yield "%s %s" % (o, a), "%s %s" % (op, args), gone, need
                    continue
            gone += int(a, 0) + 1 if o == "s_nop" else 1
            if o != "s_branch":
                todo.append((j + 1, gone))
            if target is not None:
                todo.append((target, gone))
