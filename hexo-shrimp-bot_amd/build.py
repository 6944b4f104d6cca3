"""In-tree build of the native libraries (run by ``__graft_entry__.build()``).

* ``libhexo_encoder.so`` — host C++ (g++), no GPU dependency;
* ``libmantis_hip.so`` — HIP for gfx950 (hipcc --offload-arch=gfx950);
* ``libmantis_torch.so`` — the training operators on torch's dispatcher, over
  ``libmantis_hip.so`` (g++ against the installed torch's headers);
* ``oracle/liboracle.so`` — the CPU oracle used by the tests (gcc).

Every HIP object is compiled with packed-FP32 instruction selection disabled
(``-Xclang -target-feature -Xclang -packed-fp32-ops``).
"""

from __future__ import annotations

import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
BUILD = PKG / "_build"
HIP_SOURCES = ["gather_ops.hip", "stone_attention.hip", "stone_attention_backward.hip", "hex_message.hip", "fused_linear.hip", "heads.hip",
               "attention_substage.hip", "cell_heads.hip", "latent_mix.hip", "improve.hip", "relay.hip", "attn_backward.hip", "plan.hip", "latent_broadcast.hip",
               "latent_read.hip", "latent_backward.hip", "class_order.hip", "leaf_forward.hip", "radius_stage.hip",
               "relative_attention.hip", "relative_attention_backward.hip", "policy_log_probs.hip", "residual_dropout.hip"]
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
HIP_FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    # MFMA results in VGPRs (the unified register file), not AGPRs: saves the
    # accvgpr copies between the matrix products and the softmax/epilogue math
    "-mllvm", "-amdgpu-mfma-vgpr-form",
]


def _run(cmd: list[str]) -> None:
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError(f"build step failed: {' '.join(cmd)}")


def build_encoder() -> Path:
    out = PKG / "libhexo_encoder.so"
    _run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-pthread", "-Wall",
          "-o", str(out), str(CSRC / "encoder" / "hexo_encoder.cpp")])
    return out


def build_hip() -> Path:
    BUILD.mkdir(exist_ok=True)
    objs = []

    def one(src: str) -> Path:
        obj = BUILD / (Path(src).stem + ".o")
        _run([HIPCC, *HIP_FLAGS, "-c", str(CSRC / "kernels" / src), "-o", str(obj)])
        return obj

    with ThreadPoolExecutor(max_workers=len(HIP_SOURCES)) as pool:
        objs = list(pool.map(one, HIP_SOURCES))
    out = PKG / "libmantis_hip.so"
    _run([HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", str(out), *map(str, objs)])
    return out


def build_operators() -> Path:
    import torch  # (its headers and libraries)

    home = Path(torch.__file__).resolve().parent
    rocm = Path(os.environ.get("ROCM_PATH", "/opt/rocm"))
    out = PKG / "libmantis_torch.so"
    _run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-Wno-sign-compare", "-Wno-unused-function",
          "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
          f"-I{home}/include", f"-I{home}/include/torch/csrc/api/include", "-isystem", f"{rocm}/include",
          "-o", str(out), str(CSRC / "dispatch" / "training_ops.cpp"),
          f"-L{PKG}", "-lmantis_hip", "-Wl,-rpath,$ORIGIN",
          f"-L{home}/lib", "-lc10", "-ltorch_cpu", "-ltorch", "-lc10_hip", "-ltorch_hip",
          f"-L{rocm}/lib", "-lamdhip64"])
    return out


def build_oracle() -> Path:
    _run(["make", "-s", "-C", str(ROOT / "oracle")])
    return ROOT / "oracle" / "liboracle.so"


def build_all() -> list[Path]:
    return [build_encoder(), build_hip(), build_operators(), build_oracle()]


if __name__ == "__main__":
    for p in build_all():
        print(p)
