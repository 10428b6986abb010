"""Build libsvox_hip.so for gfx950 with hipcc, in-tree (next to the sources): one object for the entry points and one
per policy of the march kernels, compiled side by side and linked; and, beside them, the host extension _host_shim.so
(host_shim.cpp: plain C++ against torch's headers, no device code).  The operators of a leaf decoder are a library of their
own, libsvox_decoder.so, with a host extension of its own, _decoder_shim.so (decoder/)."""
import os
import shutil
import subprocess
import sys
import sysconfig
import tempfile
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_NAME = "libsvox_hip.so"
SHIM_NAME = "_host_shim.so"
DECODER_LIB_NAME = "libsvox_decoder.so"
DECODER_SHIM_NAME = "_decoder_shim.so"

# -ffp-contract=off: the kernels spell their fused multiply-adds out; the compiler adds none.
# -munsafe-fp-atomics: floating-point atomicAdd becomes the hardware global_atomic_add.
# -packed-fp32-ops off: no packed fp32 instructions are generated from scalar code.
HIPCC_FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-fvisibility=hidden",
    "-ffp-contract=off", "-munsafe-fp-atomics",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
]

# (format, basis size) of every policy svox_hip.hip dispatches to (SVOX_DISPATCH_OCTREE); the longest compilations first
POLICIES = [("SH", 25), ("SG", 25), ("SH", 16), ("SG", 16), ("SH", 9), ("SG", 9), ("SH", 4), ("SG", 4), ("SH", 1), ("SG", 1),
            ("RGBA", 0)]


# the types libsvox_decoder.so has kernels for
DECODER_TYPES = ["float", "F16", "Bf16"]
DECODER_ACTIVATIONS = ["kSilu", "kGelu", "kRelu", "kSigmoid"]


def library_path():
    return os.path.join(HERE, LIB_NAME)


def _units():
    """(name, source, extra flags) of every object of libsvox_hip.so."""
    for fmt, basis in POLICIES:
        yield (f"march_{fmt.lower()}{basis}", "march_policy.hip",
               [f"-DSVOX_POLICY_FORMAT=SVOX_FORMAT_{fmt}", f"-DSVOX_POLICY_BASIS={basis}"])
    yield "march_double", "march_double.hip", []
    yield "svox_hip", "svox_hip.hip", []


def _decoder_units():
    """... and of libsvox_decoder.so."""
    for kernels in ("ffn", "norm"):
        for of in DECODER_TYPES:
            yield f"{kernels}_{of.lower()}", os.path.join("decoder", f"{kernels}_type.hip"), [f"-DSVOX_DECODER_TYPE={of}"]
    for of in DECODER_TYPES:
        for activation in DECODER_ACTIVATIONS:
            yield (f"narrow_{of.lower()}_{activation.lower()}", os.path.join("decoder", "narrow_type.hip"),
                   [f"-DSVOX_DECODER_TYPE={of}", f"-DSVOX_DECODER_ACTIVATION={activation}"])
    yield "decoder", os.path.join("decoder", "decoder.hip"), []


def _run(cmd):
    proc = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    log = "\n".join(l for l in proc.stdout.splitlines() if "packed-fp32-ops" not in l)
    if proc.returncode != 0:
        raise RuntimeError("build failed: " + " ".join(cmd) + "\n" + log)
    return log


def _shim_command(out, name=SHIM_NAME, source="host_shim.cpp"):
    import torch
    root = os.path.dirname(torch.__file__)
    includes = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
                "/opt/rocm/include", sysconfig.get_paths()["include"]]
    libs = ["c10", "c10_hip", "torch_cpu", "torch_hip", "torch", "torch_python", "dl"]
    return (["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-D__HIP_PLATFORM_AMD__",
             "-DTORCH_EXTENSION_NAME=" + name[:-3], f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
            + [f for i in includes for f in ("-isystem", i)] + [os.path.join(HERE, source), "-o", out]
            + ["-L" + os.path.join(root, "lib")] + ["-l" + name for name in libs])


def build_library(verbose=True):
    """Compile the sources into svox_amd/csrc/: libsvox_hip.so, _host_shim.so, libsvox_decoder.so and _decoder_shim.so.
    Raises on failure.  Returns the first one's path."""
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    out = library_path()
    decoder = os.path.join(HERE, DECODER_LIB_NAME)
    shims = [(os.path.join(HERE, SHIM_NAME), SHIM_NAME, "host_shim.cpp"),
             (os.path.join(HERE, DECODER_SHIM_NAME), DECODER_SHIM_NAME, os.path.join("decoder", "decoder_shim.cpp"))]
    with tempfile.TemporaryDirectory(prefix="svox_build_") as scratch:
        def compile_unit(unit):
            name, source, extra = unit
            obj = os.path.join(scratch, name + ".o")
            return obj, _run([hipcc] + HIPCC_FLAGS + extra + ["-c", "-o", obj, os.path.join(HERE, source)])

        if verbose:
            print(" ".join([hipcc] + HIPCC_FLAGS), "-c: one object per policy of the march kernels", flush=True)
        workers = int(os.environ.get("MAX_JOBS", 0)) or min(8, os.cpu_count() or 1)
        with ThreadPoolExecutor(max_workers=workers) as pool:
            host = [pool.submit(_run, _shim_command(path + ".tmp", name, source)) for path, name, source in shims]
            units, decoder_units = list(_units()), list(_decoder_units())
            made = list(pool.map(compile_unit, units + decoder_units))
            logs = [h.result() for h in host]
        for log in logs + [log for _, log in made]:
            if verbose and log.strip():
                print(log)
        objects = [obj for obj, _ in made]
        link = [hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", "-o"]
        _run(link + [out + ".tmp"] + objects[:len(units)])
        _run(link + [decoder + ".tmp"] + objects[len(units):])
    for path in [out, decoder] + [path for path, _, _ in shims]:
        os.replace(path + ".tmp", path)
    return out


if __name__ == "__main__":
    build_library()
    sys.exit(0)
