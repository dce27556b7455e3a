"""Build ``libdsw_hip.so`` in-tree with hipcc for gfx950 (cross-compiles without a GPU)."""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "csrc")
SOURCES = ["dsw_api.hip", "dsw_spmm.hip", "dsw_gemm.hip", "dsw_gemm_x3.hip", "dsw_spmm2.hip", "dsw_wgrad_x3.hip",
           "dsw_gemm_x3s.hip", "dsw_narrow.hip", "dsw_elementwise.hip", "dsw_pool.hip", "dsw_fwd3.hip", "dsw_spmm1s.hip", "dsw_bwd3d.hip",
           "dsw_rmsnorm.hip", "dsw_fp8_mix.hip", "dsw_grad_norm.hip"]
OUT = os.path.join(HERE, "libdsw_hip.so")
BINDING_SOURCE = "dsw_torch.cpp"
BINDING = os.path.join(HERE, "_dsw_torch.so")


def hipcc_path():
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", "hipcc"):
        if cand and (os.path.isabs(cand) and os.path.exists(cand) or not os.path.isabs(cand)):
            return cand
    return "hipcc"


HEADER = os.path.join(os.path.dirname(os.path.dirname(HERE)), "include", "dsw_hip.h")


def _stale(out, deps):
    return not os.path.exists(out) or any(os.path.getmtime(d) > os.path.getmtime(out) for d in deps if os.path.exists(d))


def library_stale():
    return _stale(OUT, [HEADER] + [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".hip", ".h"))])


def binding_stale():
    return _stale(BINDING, [HEADER, os.path.join(CSRC, BINDING_SOURCE)])


def needs_build():
    return library_stale() or binding_stale()


def build_binding(verbose=True):
    """Compile the tensor binding (host code only) against the installed torch's headers."""
    import sysconfig

    import torch

    root = os.path.dirname(torch.__file__)
    lib = os.path.join(root, "lib")
    inc = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
           sysconfig.get_paths()["include"], os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "include")]
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1", "-DTORCH_EXTENSION_NAME=_dsw_torch",
           *[a for d in inc for a in ("-isystem", d)], os.path.join(CSRC, BINDING_SOURCE), "-o", BINDING,
           "-L" + lib, "-lc10", "-lc10_hip", "-ltorch", "-ltorch_cpu", "-ltorch_python"]
    if verbose:
        print("[dsw build]", " ".join(cmd), flush=True)
    subprocess.run(cmd, check=True, cwd=CSRC)
    return BINDING


def build(force=False, verbose=True):
    """Compile every .hip translation unit for gfx950 (in parallel), link libdsw_hip.so, build the tensor binding."""
    if not force and not needs_build():
        return OUT
    if not force and not library_stale():
        build_binding(verbose)
        return OUT
    from concurrent.futures import ThreadPoolExecutor

    objdir = os.path.join(CSRC, "obj")
    os.makedirs(objdir, exist_ok=True)
    # -packed-fp32-ops: no v_pk_{add,mul,fma}_f32 - some forms of these instructions (the compiler makes them from ordinary
    # scalar code) have given wrong results on MI355X now and then; the host pass of hipcc warns that it does not know the feature
    flags = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
    if os.environ.get("DSW_BUILD_DIAG") == "1":      # diagnostics build: enables the DSW_* run-time switches of csrc/
        flags.append("-DDSW_DIAG")

    def compile_one(src):
        obj = os.path.join(objdir, src.replace(".hip", ".o"))
        cmd = [hipcc_path(), *flags, "-c", os.path.join(CSRC, src), "-o", obj]
        if verbose:
            print("[dsw build]", " ".join(cmd), flush=True)
        subprocess.run(cmd, check=True, cwd=CSRC)
        return obj

    with ThreadPoolExecutor(max_workers=len(SOURCES) + 1) as ex:
        binding = ex.submit(build_binding, verbose) if force or binding_stale() else None
        objs = list(ex.map(compile_one, SOURCES))
        if binding is not None:
            binding.result()
    cmd = [hipcc_path(), "--offload-arch=gfx950", "-shared", "-fPIC", "-o", OUT, *objs]
    if verbose:
        print("[dsw build]", " ".join(cmd), flush=True)
    subprocess.run(cmd, check=True, cwd=CSRC)
    return OUT


if __name__ == "__main__":
    build(force="--force" in sys.argv)
