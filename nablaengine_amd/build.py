"""Build the HIP library libnablaengine_g1.so in-tree for gfx950 (hipcc; one shared library, the C ABI of
include/nablaengine_g1.h, nablaengine_policy.h and nablaengine_memory.h), and beside it the policy operators' torch side (g++).
`python -m nablaengine_amd.build`."""
import concurrent.futures
import os
import subprocess
import sys
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libnablaengine_g1.so")
PROF_LIB = os.path.join(HERE, "libnablaengine_g1_prof.so")
TORCH_LIB, TORCH_SOURCES = os.path.join(HERE, "libnablaengine_policy_torch.so"), ["policy_torch.cpp", "policy_memory_torch.cpp"]
SOURCES = ["g1_forward.hip", "g1_adjoint.hip", "g1_order.hip", "g1_kinematics.hip", "g1_diag.hip", "g1_capi.hip",
           "policy_norm.hip", "policy_clip.hip", "policy_attend.hip", "policy_step.hip",
           "policy_scan.hip", "policy_residual.hip", "policy_paged.hip"]
ARCH = os.environ.get("NABLA_OFFLOAD_ARCH", "gfx950")
# packed FP32 instructions off (-packed-fp32-ops): the kernels are written for scalar FP32. Warnings that mark
# undefined behaviour the optimizer exploits (a non-void function falling off its end becomes unreachable code, and a
# kernel then runs into whatever follows) are errors. Machine LICM off: the kernels hold one world per wave at the
# 256-VGPR limit, and values it hoists out of the substep and Newton loops are spilled to scratch inside them.
FLAGS = ["-O3", f"--offload-arch={ARCH}", "-std=c++17", "-fPIC", "-shared", "-Xclang", "-target-feature", "-Xclang",
         "-packed-fp32-ops", "-ffp-contract=fast", "-mllvm", "-disable-machine-licm",
         "-Wno-unused-command-line-argument", "-Werror=return-type",
         "-Werror=uninitialized", "-Werror=sometimes-uninitialized", "-Werror=array-bounds"]


def flags_of(source):
    """The flags a source is compiled with. The policy operators' kernels have registers to spare, and LDS addresses that
    machine LICM keeps out of their loops."""
    policy = source.startswith("policy_")
    return [f for f in FLAGS if not (policy and f in ("-mllvm", "-disable-machine-licm")) and f != "-shared"]


def build_torch(verbose=False):
    """Compile the policy operators' torch side (C++, no device code) into TORCH_LIB."""
    import torch
    from torch.utils.cpp_extension import include_paths
    fd, tmp = tempfile.mkstemp(prefix="libnablaengine_policy_torch.", suffix=".so.tmp", dir=HERE)
    os.close(fd)
    flags = ["-O2", "-std=c++17", "-fPIC", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
             f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-Wall", "-Wno-sign-compare"]
    flags += [f"-I{p}" for p in include_paths()] + ["-I/opt/rocm/include"]
    with tempfile.TemporaryDirectory() as objects, concurrent.futures.ThreadPoolExecutor(2) as pool:
        def run(cmd):
            if verbose:
                print(" ".join(cmd))
            return subprocess.run(cmd, capture_output=True, text=True)
        objs = [os.path.join(objects, source + ".o") for source in TORCH_SOURCES]
        runs = list(pool.map(lambda o, s: run(["g++", *flags, "-c", "-o", o, os.path.join(CSRC, s)]), objs, TORCH_SOURCES))
        if all(r.returncode == 0 for r in runs):
            runs.append(run(["g++", "-shared", "-o", tmp, *objs, f"-L{os.path.join(os.path.dirname(torch.__file__), 'lib')}",
                             "-lc10", "-ltorch_cpu", "-lc10_hip", "-L/opt/rocm/lib", "-lamdhip64"]))
    if any(r.returncode for r in runs):
        os.unlink(tmp)
        sys.stderr.write("".join(r.stdout + r.stderr for r in runs if r.returncode))
        raise RuntimeError(f"g++ failed ({[r.returncode for r in runs]})")
    mask = os.umask(0)  # the temporary file is its owner's alone, and g++ keeps that
    os.umask(mask)
    os.chmod(tmp, 0o777 & ~mask)
    os.replace(tmp, TORCH_LIB)
    return TORCH_LIB


def build(verbose=False, profile=False):
    """Compile every HIP source into the library (a temporary file renamed into place: a running process that
    has the old library loaded keeps it). profile=True builds libnablaengine_g1_prof.so with the phase counters
    (-DG1_PROFILE), a measurement build."""
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    target = PROF_LIB if profile else LIB
    fd, tmp = tempfile.mkstemp(prefix="libnablaengine_g1.", suffix=".so.tmp", dir=HERE)
    os.close(fd)
    with tempfile.TemporaryDirectory() as objects, concurrent.futures.ThreadPoolExecutor(8) as pool:
        def one(source):
            obj = os.path.join(objects, source + ".o")
            cmd = [hipcc] + flags_of(source) + (["-DG1_PROFILE"] if profile else []) + ["-c", "-o", obj,
                                                                                         os.path.join(CSRC, source)]
            if verbose:
                print(" ".join(cmd))
            return obj, subprocess.run(cmd, capture_output=True, text=True)
        done = list(pool.map(one, SOURCES))
        link = [hipcc, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", tmp] + [obj for obj, _ in done]
        runs = [r for _, r in done]
        if all(r.returncode == 0 for r in runs):
            runs.append(subprocess.run(link, capture_output=True, text=True))
    if any(r.returncode for r in runs):
        os.unlink(tmp)
        sys.stderr.write("".join(r.stdout + r.stderr for r in runs if r.returncode))
        raise RuntimeError(f"hipcc failed ({[r.returncode for r in runs]})")
    os.replace(tmp, target)
    return target


if __name__ == "__main__":
    print(build(verbose=True, profile="--profile" in sys.argv))
    print(build_torch(verbose=True))
