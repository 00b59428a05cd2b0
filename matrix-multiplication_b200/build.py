"""Build the B200 GEMM library (the equivalent of the reference's ``make cuda``).

    python matrix-multiplication_b200/build.py [--verbose-ptxas]

Compiles ``csrc/*.cu`` (in parallel) for sm_100a only into ``build/b200_matmul.so``
at the repository root (the same place relative to the loader as the
reference's ``build/matmul.so``).  The CUDA runtime is linked statically and
the driver API is reached through ``cudaGetDriverEntryPoint``, so the library
loads on a machine without a GPU driver (it then fails cleanly in
``matmul_create``).
"""

from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PACKAGE = Path(__file__).resolve().parent
ROOT = PACKAGE.parent
SOURCES = sorted((PACKAGE / "csrc").glob("*.cu"))
HEADERS = sorted((PACKAGE / "csrc").glob("*.cuh")) + [ROOT / "include" / "b200_matmul.h"]
OUTPUT = ROOT / "build" / "b200_matmul.so"
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    home = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    candidate = Path(home) / "bin" / "nvcc"
    return str(candidate) if candidate.exists() else (shutil.which("nvcc") or "nvcc")


COMPILE_FLAGS = ["-O3", "-std=c++17", *ARCH_FLAGS, "-lineinfo", "-Xcompiler", "-fPIC", "-I", str(ROOT / "include")]
LINK_FLAGS = [*ARCH_FLAGS, "-shared", "-Xcompiler", "-fPIC", "-cudart", "static"]


def command(output: Path = OUTPUT, verbose_ptxas: bool = False) -> list[str]:
    """The one-step form of the build, with the flags of both of its steps (``build`` itself compiles the sources in
    parallel)."""
    cmd = [nvcc(), *COMPILE_FLAGS, *(flag for flag in LINK_FLAGS if flag not in COMPILE_FLAGS), "-o", str(output),
           *map(str, SOURCES)]
    if verbose_ptxas:
        cmd[1:1] = ["-Xptxas", "-v"]
    return cmd


def compile_command(source: Path, target: Path, verbose_ptxas: bool = False) -> list[str]:
    """One source into an object file."""
    cmd = [nvcc(), *COMPILE_FLAGS, "-c", "-o", str(target), str(source)]
    if verbose_ptxas:
        cmd[1:1] = ["-Xptxas", "-v"]
    return cmd


def link_command(objects: list[Path], output: Path) -> list[str]:
    return [nvcc(), *LINK_FLAGS, "-o", str(output), *map(str, objects)]


def up_to_date(output: Path = OUTPUT) -> bool:
    if not output.exists():
        return False
    built = output.stat().st_mtime
    return all(path.stat().st_mtime <= built for path in [*SOURCES, *HEADERS, Path(__file__)])


def _run(cmd: list[str]) -> str:
    result = subprocess.run(cmd, capture_output=True, text=True)
    if result.returncode != 0:
        raise RuntimeError(f"nvcc failed ({result.returncode}):\n{result.stdout}\n{result.stderr}")
    return result.stderr


def build(force: bool = False, verbose_ptxas: bool = False, output: Path = OUTPUT) -> Path:
    """Compile the library unless it is newer than every source; return its path."""
    if not force and not verbose_ptxas and up_to_date(output):
        return output
    output.parent.mkdir(parents=True, exist_ok=True)
    with tempfile.TemporaryDirectory(dir=output.parent) as folder:
        objects = [Path(folder) / f"{source.stem}.o" for source in SOURCES]
        tmp = Path(folder) / output.name
        with ThreadPoolExecutor(max_workers=len(SOURCES)) as pool:
            texts = list(pool.map(_run, [compile_command(s, o, verbose_ptxas) for s, o in zip(SOURCES, objects)]))
        _run(link_command(objects, tmp))
        if verbose_ptxas:
            print("\n".join(texts), file=sys.stderr)
        os.replace(tmp, output)
    return output


def main() -> int:
    parser = argparse.ArgumentParser(description=__doc__)
    parser.add_argument("--force", action="store_true")
    parser.add_argument("--verbose-ptxas", action="store_true")
    args = parser.parse_args()
    path = build(force=args.force, verbose_ptxas=args.verbose_ptxas)
    print(path)
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
