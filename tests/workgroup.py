"""Kernels of one source file on the CPU (workgroup.h): the entry points as they are, their
launches run by fibres. For what a GPU run cannot show safely: an access that another wave's
may come before or after."""

import ctypes
import re
import subprocess
from pathlib import Path

from tinyserver_amd import _build as B
from tinyserver_amd import _lib

HERE = Path(__file__).resolve().parent

# What the kernels take from tsa_common.h beside its host part and element helpers.
DEVICE = """
namespace tsa {
void set_error(const char* fmt, ...) {}
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
inline float fast_exp2(float x) { return exp2f(x); }
template <int J> inline uint32_t xor_lane32(uint32_t v, int lane) { return wg::from_lane(v, lane ^ J); }
template <int J> inline uint64_t xor_lane64(uint64_t v, int lane) { return wg::from_lane(v, lane ^ J); }
}  // namespace tsa
"""


def compiler() -> Path | None:
    for path in (Path("/opt/rocm/llvm/bin/clang++"), Path("/opt/rocm/bin/amdclang++")):
        if path.exists():
            return path
    return None


def load(source: str, tmp_path: Path, change=lambda text: text) -> ctypes.CDLL:
    """The entry points of csrc/``source``, its text as ``change`` gives it back."""
    common = (B.CSRC / "tsa_common.h").read_text().replace("#pragma once", "").replace("#include <hip/hip_runtime.h>", "")
    cut = common.index("// ------------------------------------------------------------ MFMA types --")
    text = change((B.CSRC / source).read_text()).replace('#include "tsa_common.h"', "")
    # kernel<T><<<grid, block, 0, stream>>>(args);
    text, n = re.subn(r"(\w+<T>)<<<(.+?), (dim3\([^<>]*?\)), 0, stream>>>\((.*?)\);",
                      r"wg::launch(\2, \3, [=] { \1(\4); });", text)
    assert n > 0 and "<<<" not in text
    src = tmp_path / (source + ".cpp")
    src.write_text(f'#include "workgroup.h"\n{common[:cut]}\n}}  // namespace tsa\n{DEVICE}\n{text}')
    out = tmp_path / (source + ".so")
    cmd = [str(compiler()), "-x", "c++", "-std=c++17", "-O2", "-w", "-fPIC", "-shared", f"-I{HERE}", f"-I{B.ROOT / 'include'}",
           str(src), "-o", str(out)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    assert proc.returncode == 0, proc.stderr[-3000:]
    lib = ctypes.CDLL(str(out))
    for name in re.findall(r'extern "C" \w+ (tsa_\w+)', text):
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = _lib.SIGNATURES[name]
    lib.wg_error.restype = ctypes.c_char_p
    return lib
