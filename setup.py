"""Build hook of the HIP extension: ``libmsda.so`` is compiled with hipcc for gfx950 (no torch
headers, plain C ABI) before the Python package is assembled.

    python setup.py build_hip          # just the library, in-tree
    pip install .                      # build_py runs build_hip first

Replaces the CUDA extension build the reference's container prepared for
(Containerfile:6-9 of the reference: FORCE_CUDA, TORCH_CUDA_ARCH_LIST)."""

import os
import subprocess
import sys
from pathlib import Path

from setuptools import Command, setup
from setuptools.command.build_py import build_py

ROOT = Path(__file__).resolve().parent
HIP_ARCH = "gfx950"


def hip_command(out: Path) -> list[str]:
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    return [
        hipcc, "-O3", f"--offload-arch={HIP_ARCH}", "-std=c++17", "-shared", "-fPIC",
        "-munsafe-fp-atomics", "-fno-slp-vectorize",
        "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
        "-Wall", "-Wno-unused-function", "-Wno-pass-failed",
        "-o", str(out), str(ROOT / "unipercept_amd" / "csrc" / "msda.hip"),
    ]


def torch_ops_command(out: Path) -> list[str]:
    """The torch operators over the library: host code only, against the installed PyTorch-ROCm."""
    from torch.utils import cpp_extension

    flags = ["-O2", "-std=c++17", "-shared", "-fPIC", "-Wall", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM"]
    includes = [f for d in cpp_extension.include_paths("cuda") for f in ("-isystem", d)]
    libs = [f"-L{d}" for d in cpp_extension.library_paths("cuda")]
    return [
        os.environ.get("CXX", "g++"), *flags, *includes, "-o", str(out),
        str(ROOT / "unipercept_amd" / "torch_ops" / "epilogue.cpp"), *libs,
        "-ltorch_cpu", "-lc10", "-lc10_hip",
    ]


class build_hip(Command):
    description = "compile libmsda.so with hipcc for gfx950, and libmsda_torch.so over it"
    user_options = [("force", "f", "rebuild even when the library is newer than its sources")]

    def initialize_options(self):
        self.force = False

    def finalize_options(self):
        pass

    def run(self):
        out = ROOT / "unipercept_amd" / "libmsda.so"
        deps = list((ROOT / "unipercept_amd" / "csrc").glob("*")) + [ROOT / "include" / "msda.h"]
        if not self.force and out.exists() and all(out.stat().st_mtime >= d.stat().st_mtime for d in deps):
            print(f"{out} is up to date")
        else:
            cmd = hip_command(out)
            print(" ".join(cmd))
            subprocess.run(cmd, check=True)
        # always compiled: a library of an earlier build may be another torch's, which its age does not tell
        try:
            cmd = torch_ops_command(ROOT / "unipercept_amd" / "libmsda_torch.so")
        except ModuleNotFoundError as e:
            if e.name != "torch":
                raise
            print(
                "warning: torch cannot be imported in this build environment, so libmsda_torch.so "
                "(counter_dropout, dropout_add_layer_norm, level_group_norm) is not built; "
                "`pip install --no-build-isolation .` builds it against the installed torch",
                file=sys.stderr,
            )
            return
        print(" ".join(cmd))
        subprocess.run(cmd, check=True)


class build_py_with_hip(build_py):
    def run(self):
        self.run_command("build_hip")
        super().run()


if __name__ == "__main__":
    sys.path.insert(0, str(ROOT))
    setup(cmdclass={"build_hip": build_hip, "build_py": build_py_with_hip})
