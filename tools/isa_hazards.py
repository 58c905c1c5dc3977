"""gfx950 wants one wait state between a transcendental's write (v_exp / v_rcp / v_log / v_sqrt / v_rsq / v_sin / v_cos) and a
non-transcendental VALU read of the result.  The compiler inserts it for its own instructions, but it does not look inside an
asm statement: a `v_pk_fma_f32` written as inline asm directly behind the `v_exp_f32` that feeds it reads the register's OLD
value (round 4: the first version of the backward carry pass -- 28 such pairs, 15 of 16 states wrong).

This scans the gfx950 ISA of the sources that hold asm VALU statements for that pattern.

A matrix instruction's result needs its wait states as well before any other instruction may touch it.  The compiler counts them
back over the blocks that lead to the use, but visits each block once: where a short conditional block joins another short one it has
missed the nearer way (a spill of a product one state behind the v_mfma that makes it: single elements of gradients wrong now and then).
`--mfma [library]` looks at every v_mfma of the built library along all ways out of its block.

usage: python tools/isa_hazards.py [file.s ...]      (no arguments: compile csrc/selective_scan_{fwd,bwd}_pair.hip to ISA first)
       python tools/isa_hazards.py --mfma [libvms_hip.so]
exit status 1 if a hazard was found."""
import concurrent.futures
import os
import re
import shutil
import subprocess
import sys
import tempfile

ROOT = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..")
CSRC = os.path.join(ROOT, "video-mamba-suite_amd", "csrc")
ASM_SOURCES = ("selective_scan_fwd_pair.hip", "selective_scan_bwd_pair.hip")     # grep 'asm("v_' csrc/*.hip
TRANS = re.compile(r"^\s*v_(exp|rcp|log|sqrt|rsq|sin|cos)_(f32|f16|legacy_f32)\S*\s+(v\d+)")
ASM_VALU = ("v_pk_fma_f32",)                                                     # the VALU instructions written as inline asm


def scan(path):
    """[(trans dst, consumer line)] where an ASM_VALU instruction directly follows the transcendental that writes one of its sources"""
    found, prev = [], None
    for line in open(path):
        s = line.strip()
        if not s or s[0] in ";." or s.endswith(":"):
            continue
        if prev is not None and s.startswith(ASM_VALU):
            reg = int(prev[1:])
            srcs = s.split(None, 1)[1].split(",", 1)[1]
            if any(int(a) <= reg <= int(b) for a, b in re.findall(r"v\[(\d+):(\d+)\]", srcs)):
                found.append((prev, s))
        m = TRANS.match(line)
        prev = m.group(3) if m else None
    return found


# v_mfma: wait states before its result may be read or written by anything but the next product of the same accumulator
MFMA_WAITS = {"v_mfma_f32_16x16x32_bf16": 8, "v_mfma_f32_16x16x32_f16": 8, "v_mfma_f32_16x16x4_f32": 10, "v_mfma_f32_32x32x16_bf16": 12,
              "v_mfma_f32_32x32x16_f16": 12}
LOADS = ("ds_read", "global_load", "scratch_load", "buffer_load", "flat_load")
OBJDUMP = os.environ.get("ROCM_PATH", "/opt/rocm") + "/llvm/bin/llvm-objdump"


def vgprs(operand):
    m = re.match(r"v(?:\[(\d+):(\d+)\]|(\d+)$)", operand)
    return set() if not m else {int(m[3])} if m[3] else set(range(int(m[1]), int(m[2]) + 1))


def disassembly(library):
    """{kernel: [(address, opcode, operands)]} of the library's gfx950 kernels with matrix instructions"""
    kernels = {}
    with tempfile.TemporaryDirectory(prefix="vms_isa_") as tmp:
        subprocess.check_call([OBJDUMP, "--offloading", os.path.abspath(shutil.copy(library, tmp))], cwd=tmp, stdout=subprocess.DEVNULL)
        for f in sorted(f for f in os.listdir(tmp) if "gfx950" in f):
            text = subprocess.run([OBJDUMP, "-d", os.path.join(tmp, f)], capture_output=True, text=True, check=True).stdout
            kernels |= parse_disassembly(text)
    return kernels


def parse_disassembly(text):
    kernels = {}
    for part in re.split(r"^[0-9a-f]+ (?=<.*>:$)", text, flags=re.M)[1:]:
        if "v_mfma" in part:
            name, _, lines = part.partition("\n")
            kernels[name[1:-2]] = [(int(a, 16), op, [x.strip() for x in args.split(",")] if args else [])
                                   for op, args, a in re.findall(r"^\s+(\S+) *(.*?) *// ([0-9A-F]+):", lines, flags=re.M)]
    return kernels


def scan_mfma(body):
    """[(wait states, v_mfma, the instruction that touches its result too early)] along all ways of a kernel"""
    at = {a: i for i, (a, _, _) in enumerate(body)}
    found = []
    for i, (_, op, ops) in enumerate(body):
        if not op.startswith("v_mfma"):
            continue
        need, result = MFMA_WAITS[op], vgprs(ops[0])   # (an instruction without an entry is a KeyError: add its wait states)
        best, ways = {}, [(i + 1, 0)]
        while ways:
            j, waited = ways.pop()
            while j < len(body) and waited < need and best.get(j, need) > waited:
                best[j] = waited
                a, o, args = body[j]
                if o.startswith("v_mfma"):
                    touched = (vgprs(args[1]) | vgprs(args[2])) & result
                    if not touched and (vgprs(args[0]) & result or vgprs(args[3]) == result):   # goes on in the same accumulator, or starts from it (and is held
                        break                                                                  # until it is there): its own result has its own waits
                else:
                    touched = set().union(*(vgprs(x.split()[0]) for x in (args[1:] if o.startswith(LOADS) else args) if x)) & result if args else set()
                if touched:
                    found.append((waited, f"{op} {', '.join(ops)}", f"{o} {', '.join(args)}"))
                    break
                if o == "s_endpgm":
                    break
                waited += int(args[0], 0) + 1 if o == "s_nop" else 1
                if o == "s_branch" or o.startswith("s_cbranch"):
                    n = int(args[0])
                    target = at[a + 4 + 4 * (n - 65536 if n >= 32768 else n)]
                    if o == "s_branch":
                        j = target
                        continue
                    ways.append((target, waited))
                j += 1
    return found


def main_mfma(library):
    bad = 0
    for name, body in disassembly(library).items():
        for waited, product, use in scan_mfma(body):
            bad += 1
            print(f"{name}: {product}: {use} {waited} wait states behind")
    print(f"{os.path.basename(library)}: {bad} early use(s) of a matrix instruction's result")
    return 1 if bad else 0


def to_isa(src, out):
    subprocess.check_call(["hipcc", "--offload-arch=gfx950", "-O3", "-std=c++17", "--cuda-device-only", "-S",
                           "-I" + os.path.join(ROOT, "include"), "-I" + CSRC, os.path.join(CSRC, src), "-o", out],
                          stderr=subprocess.DEVNULL)
    return out


def main(argv):
    if argv[:1] == ["--mfma"]:
        return main_mfma(argv[1] if len(argv) > 1 else os.path.join(CSRC, "..", "vms_hip", "libvms_hip.so"))
    if argv:
        files = argv
    else:
        tmp = tempfile.mkdtemp(prefix="vms_isa_")
        with concurrent.futures.ThreadPoolExecutor(len(ASM_SOURCES)) as ex:
            files = list(ex.map(lambda s: to_isa(s, os.path.join(tmp, s[:-4] + ".s")), ASM_SOURCES))
    bad = 0
    for f in files:
        h = scan(f)
        bad += len(h)
        for reg, use in h[:8]:
            print(f"{os.path.basename(f)}: {reg} written by a transcendental, read by the next instruction: {use}")
        print(f"{os.path.basename(f)}: {len(h)} hazard(s)")
    return 1 if bad else 0


if __name__ == "__main__":
    sys.exit(main(sys.argv[1:]))
