"""Build libymk.so (hand-written HIP for gfx950) in-tree with hipcc.

`python -m yolo_master_amd.build` or `__graft_entry__.build()`.  Objects are cached by
source mtime and compile flags under yolo_master_amd/csrc/_obj/; the shared library lands next to this file
so that it travels with the tree and is the one the tests load.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
OBJ = CSRC / "_obj"
LIB = HERE / "libymk.so"
# The same sources compiled a second time with the 16-bit element format = IEEE binary16 (-DYMK_H16_F16, csrc/ymk_common.h): same
# C-ABI, loaded side by side by _lib.py for torch.float16 tensors (the reference's `half=True` mode).
VARIANTS = {"bf16": (OBJ, LIB, []), "f16": (CSRC / "_obj_f16", HERE / "libymk_f16.so", ["-DYMK_H16_F16"])}
ARCH = "gfx950"
# Packed fp32 instructions stay out of all kernels (some of their forms have given wrong results on this hardware): fp32 pair arithmetic in the sources
# (csrc/dwconv.hip) compiles to two instructions.  The detector's step takes the same time either way (4.87 ms, two runs of each differ by 1.5 %).
NO_PACKED_FP32 = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
# files whose arithmetic must not be contracted into FMAs (bit-exact NMS / decode)
NO_CONTRACT = {"nms.hip", "elementwise.hip", "post.hip", "preproc.hip"}
TOKEN_SOURCES = ["rmsnorm.hip", "tokens.hip", "expert.hip"]   # norms, tokens by expert, the experts' product (include/ymk_tokens.h)
SOURCES = ["capi.hip", "conv.hip", "dwconv.hip", "mlp.hip", "stem2.hip", "c3k2f.hip", "detcls.hip", "esmoe.hip", "attn.hip", "elementwise.hip", "nms.hip",
           "mixture.hip", "mixattn.hip",   # config-5 rows, first implementation (include/ymk_mixture.h)
           *TOKEN_SOURCES,
           "conv_glds.hip", "post.hip", "preproc.hip"]   # LDS-DMA tiled convolution core, box rescaling / validation matching, letterbox (include/ymk_next.h)
HEADERS = ["ymk_common.h", "igemm.h", "glds.h", "rows.h", "../../include/ymk.h", "../../include/ymk_mixture.h", "../../include/ymk_next.h", "../../include/ymk_tokens.h"]


def _hipcc() -> str:
    for cand in (shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found: libymk cannot be built (ROCm toolchain required)")


def _flags(src: str, defs: list) -> list:
    """What hipcc is told of one source, without paths."""
    flags = [f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC", *defs, *NO_PACKED_FP32]
    if src in NO_CONTRACT:
        flags.append("-ffp-contract=off")
    if src in ("post.hip", "preproc.hip"):   # bit-exact box rescaling divides by the gain: IEEE division (hipcc's default, stated explicitly)
        flags.append("-fhip-fp32-correctly-rounded-divide-sqrt")
    return flags


def source_hash(tokens: bool = False) -> str:
    """sha256 (16 hex digits) over the detector's kernel sources (or the token operators'), their shared headers and the flags that each is compiled
    with, comments aside (they quote what a profile measured): committed rocprofv3 summaries carry it, so that a profile is only ever quoted for the kernels it was collected on (bench.py
    `roofline.traffic`, `families[].sq`)."""
    import hashlib
    import re

    h = hashlib.sha256()
    sources, headers = (TOKEN_SOURCES, ["ymk_common.h", "rows.h", "glds.h"]) if tokens else (set(SOURCES) - set(TOKEN_SOURCES), ["ymk_common.h", "igemm.h", "glds.h"])
    for f in sorted(sources) + headers:
        h.update(f.encode())
        code = re.sub(r"//[^\n]*|/\*.*?\*/", "", (CSRC / f).read_text(), flags=re.S)
        h.update("\n".join(line.rstrip() for line in code.splitlines() if line.strip()).encode())
        if f.endswith(".hip"):
            h.update(" ".join(_flags(f, [])).encode())
    return h.hexdigest()[:16]


def _compile_cmd(hipcc: str, src: str, obj: Path, defs: list) -> list:
    return [hipcc, *_flags(src, defs), "-c", str(CSRC / src), "-o", str(obj)]


def _stale(src: str, obj: Path, flags: list, headers: float) -> bool:
    """The object is older than its source or the shared headers, or was compiled with other flags (kept beside it)."""
    note = obj.with_suffix(".flags")
    return not obj.exists() or obj.stat().st_mtime < max((CSRC / src).stat().st_mtime, headers) or not note.exists() or note.read_text() != " ".join(flags)


def build(force: bool = False, verbose: bool = True, variants=("bf16", "f16")) -> Path:
    """Compile what is stale (objects are cached by mtime against their source and the shared headers, and by their flags) for every variant, up to
    $YMK_BUILD_JOBS (default: all cores) hipcc processes at a time, then link each variant's shared object."""
    from concurrent.futures import ThreadPoolExecutor

    hipcc = _hipcc()
    hdr_m = max((CSRC / h).resolve().stat().st_mtime for h in HEADERS)
    jobs, relink = [], set()
    for v in variants:
        obj_dir, lib, defs = VARIANTS[v]
        obj_dir.mkdir(exist_ok=True)
        for src in SOURCES:
            o = obj_dir / src.replace(".hip", ".o")
            flags = _flags(src, defs)
            if not force and not _stale(src, o, flags, hdr_m):
                continue
            jobs.append((_compile_cmd(hipcc, src, o, defs), o.with_suffix(".flags"), " ".join(flags)))
            relink.add(v)
        if force or not lib.exists():
            relink.add(v)

    def run(cmd):
        if verbose:
            print("[ymk build]", " ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)

    def compile_one(job):
        cmd, note, flags = job
        note.unlink(missing_ok=True)   # a compilation that fails leaves the object stale
        run(cmd)
        note.write_text(flags)

    if jobs:
        with ThreadPoolExecutor(max_workers=int(os.environ.get("YMK_BUILD_JOBS", os.cpu_count() or 4))) as ex:
            list(ex.map(compile_one, jobs))
    for v in variants:
        obj_dir, lib, _ = VARIANTS[v]
        if v in relink:
            # -Bsymbolic + hidden-by-default template instantiations are not needed: ctypes loads each library RTLD_LOCAL, so the two
            # variants' identically named symbols never meet
            run([hipcc, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-Wl,-Bsymbolic", "-o", str(lib), *[str(obj_dir / s.replace(".hip", ".o")) for s in SOURCES]])
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv)
    print(LIB)
