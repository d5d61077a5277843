"""Results of matrix instructions that are read too early, found in the gfx950 assembly of our own kernels.

gfx950 does not hold back an instruction that reads the registers an MFMA is still writing: the compiler has to leave 2 + passes wait states
(f32 operands) or 4 + passes (16- and 8-bit ones).  hipcc counts them along one path only where two branches of different length meet behind
the MFMA, and then leaves too few on the shorter one.  This walks all paths and takes the shortest.

usage: python tools/mfma_waits.py a.s ...  -> one line a kernel, exit status 1 if any reads too early"""
import heapq
import re
import sys

PASSES = {"32x32x16": 8, "16x16x32": 4, "32x32x8": 16, "16x16x16": 8, "32x32x4": 16, "32x32x2": 16, "16x16x4": 8, "16x16x128": 8, "32x32x64": 16}
MEMORY = ("ds_", "global_", "buffer_", "flat_", "scratch_")


def registers(text):
    out = set()
    for m in re.finditer(r"\b([av])\[(\d+):(\d+)\]|\b([av])(\d+)\b", text):
        if m.group(1):
            out |= {(m.group(1), i) for i in range(int(m.group(2)), int(m.group(3)) + 1)}
        else:
            out.add((m.group(4), int(m.group(5))))
    return out


def functions(path):
    """{name: ([(opcode, [operands])], {label: index})}"""
    out, name = {}, None
    with open(path) as f:
        for line in f:
            line = line.split(";")[0].rstrip()
            m = re.match(r"([A-Za-z_.$][\w.$]*):", line)
            if m and m.group(1).startswith(".Lfunc_end"):
                name = None
            elif m and m.group(1).startswith(".L"):
                if name:
                    out[name][1][m.group(1)] = len(out[name][0])
            elif m:
                name = m.group(1)
                out[name] = ([], {})
            elif name and line[:1] in " \t" and line.strip() and not line.strip().startswith("."):
                op, _, rest = line.strip().partition(" ")
                op, _, more = op.partition("\t")
                out[name][0].append((op, [x.strip() for x in re.split(r",\s*(?![^\[]*\])", more + rest)]))
    return out


def early(code, labels):
    """[(index of the MFMA, index of the reader, wait states, needed)]"""
    found = []
    for k, (op, args) in enumerate(code):
        if not op.startswith("v_mfma"):
            continue
        shape = re.search(r"\d+x\d+x\d+", op).group()
        narrow = re.search(r"f16|bf8|fp8|i8|f8", op.split(shape)[1])
        need, dst = PASSES[shape] + (4 if narrow else 2), registers(args[0])
        best, todo = {k + 1: 0}, [(0, k + 1)]
        while todo:
            d, i = heapq.heappop(todo)
            if d > best[i] or d >= need or i >= len(code):
                continue
            o, a = code[i]
            if o.startswith("v_mfma"):
                if registers(",".join(a[1:3])) & dst:
                    found.append((k, i, d, need))
                if registers(a[0]) >= dst:
                    continue                                 # the sum goes on, in order
            elif o.startswith("v_") or o.startswith(MEMORY):
                # (what a load brings arrives long after)
                loads = o.startswith(MEMORY) and ("load" in o or "read" in o)
                if registers(",".join(a[1:] if loads else a)) & dst:
                    found.append((k, i, d, need))
                    continue
            if o == "s_endpgm":
                continue
            d += int(a[0].split()[0], 0) + 1 if o == "s_nop" else 1
            ways = [labels.get(a[0])] if o == "s_branch" else [labels.get(a[0]), i + 1] if o.startswith("s_cbranch") else [i + 1]
            for n in ways:
                if n is not None and d < best.get(n, need):
                    best[n] = d
                    heapq.heappush(todo, (d, n))
    return found


if __name__ == "__main__":
    total = 0
    for path in sys.argv[1:]:
        for name, (code, labels) in functions(path).items():
            count = sum(op.startswith("v_mfma") for op, _ in code)
            if count:
                bad = early(code, labels)
                total += len(bad)
                print(name, "mfma", count, "early", len(bad), [(code[k][0], code[i][0], d, n) for k, i, d, n in bad[:3]])
    sys.exit(1 if total else 0)
