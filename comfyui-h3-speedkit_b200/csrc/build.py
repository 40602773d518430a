"""Build the sm_100a kernel library in-tree and write its manifest.

Output: ``h3_speedkit/_native/libh3sk_b200.so`` plus one symlink per library
name the reference loads (``norm.so``, ``residual.so``, ``convrot.so``, ``fc1.so``, ``gate.so``, ``qkv.so``,
``sample.so``, ``anchor.so``)
and ``build.json`` in the reference's manifest schema
(tools/build_kernels.py:41-63 of H3 SpeedKit: schema, kernels[name].sha256 ...).

The quantiser translation units are compiled with ``--use_fast_math`` exactly
as the reference compiles its norm/convrot kernels (tools/build_kernels.py:32-34),
because the quantiser's division must be the same operation; the GEMM unit is
compiled without it and spells every epilogue rounding explicitly.  The QKV head
epilogue is compiled without it and the K anchor detector and the INT8
attention with it, as the reference compiles its qkv/sample, anchor and dense
units (tools/build_kernels.py:30-37).  ``h3sk_torch.so`` beside the library is the
PyTorch binding of the operators that are called once per token (``bind.cpp``); the
manifest's ``binding`` names the library, the torch and the Python it was made for.
"""
from __future__ import annotations

import argparse
import hashlib
import json
import os
import platform
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from importlib import metadata
from pathlib import Path

CSRC = Path(__file__).resolve().parent
PKG = CSRC.parent
NATIVE = PKG / "h3_speedkit" / "_native"
BUILD = PKG / "_build"
LIB_NAME = "libh3sk_b200.so"
BINDING_NAME = "h3sk_torch.so"
ALIASES = ("norm", "residual", "convrot", "fc1", "gate", "qkv", "sample", "anchor", "dense")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON = ["-std=c++17", "-O3", "-DNDEBUG", "-lineinfo", "-Xcompiler", "-fPIC", "-Xptxas", "-v",
          "--expt-relaxed-constexpr"]
UNITS = (
    ("norm_quant.cu", ["--use_fast_math", "-DH3SK_QUANT_FAST_MATH"]),
    ("convrot_quant.cu", ["--use_fast_math", "-DH3SK_QUANT_FAST_MATH"]),
    ("int8_gemm.cu", []),
    ("qkv_quant.cu", []),
    ("anchor.cu", ["--use_fast_math"]),
    ("attention.cu", ["--use_fast_math"]),
    ("rms_quant.cu", []),
    ("rope.cu", []),
    ("masked_attention.cu", []),
    ("masked_attention_fp16.cu", []),
)


def sha256(path: Path) -> str:
    return hashlib.sha256(path.read_bytes()).hexdigest()


def nvcc_path(explicit: str | None = None) -> str:
    for candidate in (explicit, shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if candidate and Path(candidate).exists():
            return candidate
    raise RuntimeError("nvcc not found; the CUDA toolkit is required to build the sm_100a library")


def run(cmd: list[str]) -> subprocess.CompletedProcess:
    return subprocess.run(cmd, text=True, capture_output=True)


def hosts() -> dict:
    """What the binding is compiled against; another of either needs another binding."""
    return {"torch": metadata.version("torch"), "python": platform.python_version()}


def up_to_date() -> bool:
    built = (NATIVE / LIB_NAME, NATIVE / BINDING_NAME)
    if not all(p.exists() for p in built) or not (NATIVE / "build.json").exists():
        return False
    newest = max(p.stat().st_mtime for p in [q for kind in ("*.cu", "*.cuh", "*.h", "*.cpp") for q in CSRC.glob(kind)]
                 + [PKG.parent / "include" / "h3sk_b200.h", Path(__file__)])
    if min(p.stat().st_mtime for p in built) < newest:
        return False
    binding = json.loads((NATIVE / "build.json").read_text()).get("binding", {})
    return all(binding.get(name) == version for name, version in hosts().items())


def binding_command(library: Path, out: Path) -> list[str]:
    """The command that compiles bind.cpp against this interpreter's torch and `library`."""
    import torch
    root = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc_path()).resolve().parents[1]
    includes = [root / "include", root / "include/torch/csrc/api/include", sysconfig.get_paths()["include"], cuda / "include"]
    return ["g++", "-std=c++17", "-O2", "-fPIC", "-shared", "-DNDEBUG", "-fvisibility=hidden",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *(f"-I{p}" for p in includes),
            str(CSRC / "bind.cpp"), "-o", str(out), f"-L{root / 'lib'}", "-ltorch_python", "-ltorch", "-ltorch_cpu",
            "-ltorch_cuda", "-lc10", "-lc10_cuda", f"-L{library.parent}", f"-l:{library.name}", "-Wl,-rpath,$ORIGIN"]


def build(nvcc: str | None = None, force: bool = False, quiet: bool = True) -> Path:
    """Build the library and the binding, and put both in place only when both are there."""
    if not force and up_to_date():
        return NATIVE / LIB_NAME
    nvcc = nvcc_path(nvcc)
    BUILD.mkdir(parents=True, exist_ok=True)
    NATIVE.mkdir(parents=True, exist_ok=True)
    version = subprocess.check_output([nvcc, "--version"], text=True)
    manifest = {"schema": 1, "status": "building", "target": "sm_100a", "nvcc": version, "kernels": {}}
    objects, logs, commands = [], [], {}

    def done(what, cmd, result):
        logs.append(f"$ {' '.join(cmd)}\n{result.stdout}{result.stderr}")
        if result.returncode:
            (NATIVE / "build.log").write_text("\n".join(logs))
            raise RuntimeError(f"{what}:\n{result.stderr[-6000:]}")

    for source, extra in UNITS:
        src = CSRC / source
        commands[source] = [nvcc, *COMMON, *ARCH, *extra, "-c", str(src), "-o", str(BUILD / (src.stem + ".o"))]
        objects.append(BUILD / (src.stem + ".o"))
    with ThreadPoolExecutor(os.cpu_count() or 1) as pool:
        results = list(pool.map(run, commands.values()))
    for (source, cmd), result in zip(commands.items(), results):
        done(f"nvcc failed on {source}", cmd, result)
    lib, binding = BUILD / LIB_NAME, BUILD / BINDING_NAME
    link = [nvcc, *ARCH, "-shared", "-Xcompiler", "-fPIC", *map(str, objects), "-o", str(lib)]
    done("link failed", link, run(link))
    bind = binding_command(lib, binding)
    done("g++ failed on bind.cpp", bind, run(bind))
    # an interruption from here on leaves no manifest, so that the next build starts again
    (NATIVE / "build.json").unlink(missing_ok=True)
    os.replace(lib, NATIVE / LIB_NAME)
    os.replace(binding, NATIVE / BINDING_NAME)
    lib, binding = NATIVE / LIB_NAME, NATIVE / BINDING_NAME
    (NATIVE / "build.log").write_text("\n".join(logs))
    digest = sha256(lib)
    manifest["binding"] = {"source": "csrc/bind.cpp", "source_sha256": sha256(CSRC / "bind.cpp"), "command": bind,
                           "file": BINDING_NAME, "sha256": sha256(binding), "library_sha256": digest, **hosts()}
    sources = {"norm": "norm_quant.cu", "residual": "norm_quant.cu", "convrot": "convrot_quant.cu",
               "fc1": "int8_gemm.cu", "gate": "int8_gemm.cu", "qkv": "qkv_quant.cu", "sample": "qkv_quant.cu",
               "anchor": "anchor.cu", "dense": "attention.cu"}
    for name in ALIASES:
        alias = NATIVE / (name + ".so")
        if alias.is_symlink() or alias.exists():
            alias.unlink()
        alias.symlink_to(LIB_NAME)
        src = CSRC / sources[name]
        manifest["kernels"][name] = {"source": f"csrc/{sources[name]}", "source_sha256": sha256(src),
                                     "exit_code": 0, "command": commands[sources[name]],
                                     "library": LIB_NAME, "sha256": digest}
    manifest["status"] = "compiled; numerical validation required"
    (NATIVE / "build.json").write_text(json.dumps(manifest, indent=2) + "\n")
    if not quiet:
        print(f"built {lib} ({lib.stat().st_size} bytes)")
    return lib


def main() -> int:
    parser = argparse.ArgumentParser(description=__doc__)
    parser.add_argument("--nvcc")
    parser.add_argument("--force", action="store_true")
    args = parser.parse_args()
    build(args.nvcc, force=args.force, quiet=False)
    return 0


if __name__ == "__main__":
    sys.exit(main())
