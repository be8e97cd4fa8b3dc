"""Build libsemseg_hip.so (gfx950) in-tree with hipcc.  No torch involvement: the library is a plain
C-ABI shared object (see include/semseg_hip.h)."""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(CSRC, "libsemseg_hip.so")
SOURCES = ["conv_igemm.hip", "conv_wgrad.hip", "stem.hip", "bn.hip", "pool_interp.hip", "ce_head.hip", "psamask.hip",
           "psa_ops.hip", "infer.hip", "optim.hip", "augment.hip", "winograd.hip", "gemm_bf16split.hip", "xchg.hip", "plan.hip", "class_logprobs.hip", "distill.hip"]
HEADER = os.path.join(HERE, "..", "include", "semseg_hip.h")
THUNKS = os.path.join(CSRC, "plan_thunks.inc")
# -packed-fp32-ops: no v_pk_add / mul / fma_f32 — some of their forms have given wrong results on this hardware now and then, with no
# error (hipcc's host pass warns that it does not know the feature: harmless)
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-munsafe-fp-atomics", "-fPIC", "-shared",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


OBJ_DIR = os.path.join(CSRC, "build")          # git-ignored; objects are an incremental-build cache only


def _deps(src):
    """The source, EVERY header of csrc/ (a changed internal prototype must not link against stale cached objects) and the C ABI."""
    import glob
    return [os.path.join(CSRC, src)] + sorted(glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.inc"))) + \
        [os.path.join(HERE, "..", "include", "semseg_hip.h")]


def parse_header_c(path=HEADER):
    """[(name, return type, [(C type text, argument name), ...])] of every entry point include/semseg_hip.h declares."""
    import re
    src = re.sub(r"/\*.*?\*/", "", open(path).read(), flags=re.S)
    out = []
    for m in re.finditer(r"\b(int|size_t)\s+(semseg_\w+)\s*\(([^)]*)\)\s*;", src):
        args = []
        for a in m.group(3).split(","):
            a = " ".join(a.split())
            if not a or a == "void":
                continue
            mm = re.match(r"^(.*?)(\w+)$", a)
            args.append((mm.group(1).strip(), mm.group(2)))
        out.append((m.group(2), m.group(1), args))
    return out


def thunks_text():
    """csrc/plan_thunks.inc: one call thunk per `int semseg_*(...)` entry point of the header, decoding a row of 64-bit slots
    (pointers and integers by value, float / double by bit pattern) into the call — what semseg_plan_replay walks (plan.hip)."""
    lines = ["// GENERATED by semseg_amd/build.py (thunks_text) from include/semseg_hip.h — do not edit; tests/test_plan_cpu.py checks it is current.",
             "// One thunk per C-ABI entry point: slots -> typed call.", ""]
    names = []
    for name, ret, args in parse_header_c():
        if ret != "int" or name.startswith("semseg_plan_"):
            continue
        conv = []
        for i, (ty, _) in enumerate(args):
            if "*" in ty or ty == "hipStream_t":
                conv.append("reinterpret_cast<%s>(static_cast<uintptr_t>(s[%d]))" % (ty, i))
            elif ty == "float":
                conv.append("slot_f32(s[%d])" % i)
            elif ty == "double":
                conv.append("slot_f64(s[%d])" % i)
            else:
                conv.append("static_cast<%s>(s[%d])" % (ty, i))
        lines.append("static int thunk_%s(const unsigned long long* s) {\n  (void)s;\n  return %s(%s);\n}"
                     % (name, name, ",\n      ".join(conv)))
        names.append((name, len(args)))
    lines.append("")
    lines.append("static const PlanThunk PLAN_THUNKS[] = {")
    for name, n in names:
        lines.append('  {"%s", thunk_%s, %d},' % (name, name, n))
    lines.append("};")
    return "\n".join(lines) + "\n"


def gen_thunks():
    text = thunks_text()
    try:
        if open(THUNKS).read() == text:
            return False
    except OSError:
        pass
    with open(THUNKS, "w") as f:
        f.write(text)
    return True


def _tag(defines=()):
    """Of the flags and defines an object was compiled with: part of its cached name."""
    import hashlib
    h = hashlib.sha1(" ".join(FLAGS + sorted(defines)).encode()).hexdigest()[:8]
    return h if defines else "base-" + h


def _linked_sources():
    """The flags' tag and the names of the sources the library on disk was linked from (written next to it at link time)."""
    try:
        return open(LIB + ".sources").read().split()
    except OSError:
        return []


def needs_build():
    if not os.path.exists(LIB) or _linked_sources() != [_tag()] + [s for s in SOURCES if os.path.exists(os.path.join(CSRC, s))]:
        return True
    t = os.path.getmtime(LIB)
    return any(os.path.getmtime(d) > t for s in SOURCES for d in _deps(s) if os.path.exists(d))


def build(force=False, verbose=False, defines=(), out=None):
    """One hipcc -c per source, in parallel, then one link.  Objects are cached per (source, defines) under csrc/build/ so
    that touching one kernel file rebuilds that file only (conv_igemm.hip and conv_wgrad.hip take about a minute each).  `defines` / `out`
    build a VARIANT library for A/B runs (scripts/; selected with SEMSEG_HIP_LIB), never the product."""
    out = out or LIB
    gen_thunks()      # before the staleness check: a header edit changes plan_thunks.inc, which plan.hip includes
    if not force and not defines and out == LIB and not needs_build():
        return LIB
    from concurrent.futures import ThreadPoolExecutor
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    os.makedirs(OBJ_DIR, exist_ok=True)
    tag = _tag(defines)
    cflags = [f for f in FLAGS if f != "-shared"] + ["-D" + d for d in defines]
    jobs = []
    for src in SOURCES:
        if not os.path.exists(os.path.join(CSRC, src)):
            continue
        obj = os.path.join(OBJ_DIR, "%s.%s.o" % (src, tag))
        stale = force or not os.path.exists(obj) or any(os.path.getmtime(d) > os.path.getmtime(obj) for d in _deps(src))
        jobs.append((src, obj, stale))

    def compile_one(job):
        src, obj, stale = job
        if stale:
            import time
            t0 = time.time()
            cmd = [hipcc] + cflags + ["-c", os.path.join(CSRC, src), "-o", obj + ".tmp"]
            if verbose:
                print(" ".join(cmd), file=sys.stderr)
            subprocess.check_call(cmd)
            os.replace(obj + ".tmp", obj)
            # the object is as old as the moment its compile STARTED: a source edited while hipcc was running (its host and
            # device passes read the file separately) is newer than the object and gets rebuilt next time
            os.utime(obj, (t0, t0))
        return obj
    with ThreadPoolExecutor(max_workers=min(8, len(jobs))) as ex:
        objs = list(ex.map(compile_one, jobs))
    cmd = [hipcc, "--offload-arch=gfx950", "-fPIC", "-shared"] + objs + ["-o", out]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    subprocess.check_call(cmd)
    with open(out + ".sources", "w") as f:
        f.write("\n".join([tag] + [j[0] for j in jobs]) + "\n")
    return out


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
