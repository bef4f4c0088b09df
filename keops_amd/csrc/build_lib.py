"""Build libkeops_hip.so (host C++ + embedded HIP kernel templates).

Usage:  python keops_amd/csrc/build_lib.py [--force]

Step 1 packs the hand-written kernel templates of csrc/kernels/*.h into kernels_embedded.inc
(raw string literals) so that the shared library can hand them to hiprtc as in-memory headers.
Step 2 compiles keops_static.hip (the device code that lives in the library itself: static scratch
buffer, fill, conversion and range-table kernels) and sequence/*.hip (the sequence operators) with hipcc for gfx950
and keops_hip.cpp with the host compiler, and links them into libkeops_hip.so next to this file, against the HIP runtime and hiprtc of the ROCm
installation (ROCM_PATH, default /opt/rocm).
Step 3 builds libkeops_calibrate.so from keops_calibrate.hip: the loop-only calibration kernels of the benchmark,
kept out of the product library.
"""
import glob
import hashlib
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
LIB = os.path.join(HERE, "libkeops_hip.so")
CALIB_LIB = os.path.join(HERE, "libkeops_calibrate.so")


def kernel_headers():
    return sorted(glob.glob(os.path.join(HERE, "kernels", "*.h")))


def templates_digest():
    h = hashlib.sha256()
    for path in kernel_headers() + [os.path.join(HERE, f) for f in ("keops_hip.cpp", "keops_static.hip", "keops_static.h", "keops_calibrate.hip", "keops_calibrate.h")]:
        h.update(open(path, "rb").read())
    return h.hexdigest()


def sequence_sources():
    return sorted(glob.glob(os.path.join(HERE, "sequence", "*.hip")))


def library_digest():
    """Of everything libkeops_hip.so is built from (the templates' digest alone is part of the kernel cache's key)."""
    h = hashlib.sha256(templates_digest().encode())
    for path in sequence_sources() + [os.path.join(HERE, "sequence", "keops_seq.h"),
                                      os.path.join(HERE, "..", "..", "include", "keops_hip.h")]:
        h.update(open(path, "rb").read())
    return h.hexdigest()


def write_embedded():
    out = ["// generated by build_lib.py from csrc/kernels/*.h - do not edit", "static const EmbeddedHeader keops_embedded_headers[] = {"]
    for path in kernel_headers():
        text = open(path).read()
        assert ')KEOPSRAW"' not in text
        # split long literals: some compilers cap a single string literal at 64 KiB
        chunks = [text[i : i + 12000] for i in range(0, len(text), 12000)]
        lit = "\n".join(f'R"KEOPSRAW({c})KEOPSRAW"' for c in chunks)
        out.append(f'  {{"{os.path.basename(path)}",\n{lit}}},')
    out.append("  {nullptr, nullptr}};")
    out.append(f'static const char* keops_templates_digest = "{templates_digest()}";')
    with open(os.path.join(HERE, "kernels_embedded.inc"), "w") as f:
        f.write("\n".join(out) + "\n")


def build(force=False):
    stamp = os.path.join(HERE, ".libkeops_hip.digest")
    digest = library_digest()
    if not force and os.path.exists(LIB) and os.path.exists(CALIB_LIB) and os.path.exists(stamp) and open(stamp).read() == digest:
        return LIB
    write_embedded()
    hipcc = os.path.join(ROCM, "bin", "hipcc")
    arch = os.environ.get("KEOPS_HIP_ARCH", "gfx950")
    static_o, host_o = os.path.join(HERE, "keops_static.o"), os.path.join(HERE, "keops_hip.o")
    # packed FP32 instructions are kept out of every kernel of this library
    flags = [f"--offload-arch={arch}", "-O3", "-std=c++17", "-fPIC", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
             "-Wno-unused-command-line-argument"]
    quiet = subprocess.DEVNULL if not os.environ.get("KEOPS_BUILD_VERBOSE") else None
    sequence_o = [os.path.splitext(path)[0] + ".o" for path in sequence_sources()]
    compilers = [subprocess.Popen([hipcc, *flags, "-c", path, "-o", obj], stderr=quiet)
                 for path, obj in zip([os.path.join(HERE, "keops_static.hip"), *sequence_sources()], [static_o, *sequence_o])]
    compilers.append(subprocess.Popen([hipcc, *flags, "-shared", os.path.join(HERE, "keops_calibrate.hip"), "-o", CALIB_LIB],
                                      stderr=quiet))
    compilers.append(subprocess.Popen([os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-Wall", "-D__HIP_PLATFORM_AMD__",
                                       f"-I{ROCM}/include", "-c", os.path.join(HERE, "keops_hip.cpp"), "-o", host_o]))
    codes = [(p.wait(), p.args) for p in compilers]
    for code, args in codes:
        if code != 0:
            raise subprocess.CalledProcessError(code, args)
    subprocess.run([hipcc, "-shared", "-fPIC", host_o, static_o, *sequence_o, "-o", LIB, f"-L{ROCM}/lib", "-lamdhip64", "-lhiprtc",
                    f"-Wl,-rpath,{ROCM}/lib"], check=True)
    with open(stamp, "w") as f:
        f.write(digest)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv))
