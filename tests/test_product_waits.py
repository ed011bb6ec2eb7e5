"""Instructions that are written out (fg_block.h) and read results of the matrix cores wait for them: the compiler counts wait states between a product and its
reader for its own instructions only.  Read from assembly of kernels built here, without a GPU."""
import os
import re
import shutil
import subprocess

import pytest

from featgraph_amd import build

# wait states between a product and an instruction that reads its result, as the compiler keeps them (test_the_compilers_own_waits)
NEEDED = {"v_mfma_f32_16x16x32_bf16": 8, "v_mfma_f32_16x16x32_f16": 8, "v_mfma_f32_16x16x4_f32": 10}

KERNELS = """
#include "fg_block.h"
using namespace fg::block;
template <typename T> __device__ void products(const T *p, f32x4 &x, f32x4 &y) {
    const auto a = load8(p + threadIdx.x * 8), b = load8(p + 1024 + threadIdx.x * 8);
    x = y = f32x4{0.f, 0.f, 0.f, 0.f};
    x = mma(a, b, x);
    y = mma(b, a, y);
}
#define KERNELS(T, NAME) \\
    extern "C" __global__ void largest_##NAME(const T *p, float *o) { f32x4 x, y; products(p, x, y); o[threadIdx.x] = largest_of_rows(largest(x, y)); } \\
    extern "C" __global__ void other_##NAME(const T *p, float *o) { f32x4 x, y; products(p, x, y); o[threadIdx.x] = largest(y, x) - largest(x, x); } \\
    extern "C" __global__ void plain_##NAME(const T *p, float *o) { f32x4 x, y; products(p, x, y); o[threadIdx.x] = y[1] * x[3]; }
KERNELS(__bf16, bf16)
KERNELS(_Float16, f16)
KERNELS(float, f32)
"""


def _registers(operand):
    one, many = re.fullmatch(r"v(\d+)", operand), re.fullmatch(r"v\[(\d+):(\d+)\]", operand)
    return {int(one.group(1))} if one else set(range(int(many.group(1)), int(many.group(2)) + 1)) if many else set()


def shortest_waits(lines):
    """{(kind of product, reader): least wait states between a product and the first reader of its result}, along the text."""
    at, pending, found = 0, {}, {}
    for line in lines:
        line = line.split("//")[0].split(";")[0].strip()
        if not re.match(r"[sv]_|ds_|global_|buffer_|flat_", line):
            continue
        name, _, rest = line.partition(" ") if " " in line else line.partition("\t")
        name, operands = name.strip(), [x.strip() for x in rest.strip().split(",")]
        mfma = name.startswith("v_mfma")
        if name.startswith("v_") and not mfma:
            for reg in set().union(*[_registers(x) for x in operands[1:]] or [set()]):
                if reg in pending:
                    kind, when = pending.pop(reg)
                    key = kind, name
                    found[key] = min(found.get(key, 1 << 30), at - when - 1)
        for reg in _registers(operands[0]) if name.startswith("v_") else ():
            pending.pop(reg, None)
            if mfma:
                pending[reg] = name, at
        at += int(operands[0], 0) + 1 if name == "s_nop" else 1
    return found


@pytest.fixture(scope="module")
def assembly(tmp_path_factory):
    try:
        hipcc = build._hipcc()
    except RuntimeError:
        pytest.skip("no compiler")
    folder = tmp_path_factory.mktemp("waits")
    (folder / "k.hip").write_text(KERNELS)
    subprocess.run([hipcc] + build.HIP_FLAGS + ["-I", build.CSRC, "-x", "hip", "--cuda-device-only", "-S", str(folder / "k.hip"), "-o", str(folder / "k.s")],
                   check=True, capture_output=True)
    found = {}
    for part in re.split(r"^(?=\w+:\s+; @)", (folder / "k.s").read_text(), flags=re.M)[1:]:
        found[part.split(":")[0]] = part.split(".section")[0].splitlines()
    return found


@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
def test_the_compilers_own_waits(assembly, name):
    waits = shortest_waits(assembly["plain_" + name])
    assert waits and all(states >= NEEDED[kind] for (kind, _), states in waits.items()), waits
    assert min(waits.values()) == NEEDED[next(iter(waits))[0]]


@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("kernel", ["largest_", "other_"])
def test_the_largest_of_products_waits_for_all_of_them(assembly, kernel, name):
    waits = shortest_waits(assembly[kernel + name])
    assert any(reader == "v_max3_f32" for _, reader in waits), waits
    assert all(states >= NEEDED[kind] for (kind, _), states in waits.items()), waits


def test_kernels_of_the_library(tmp_path):
    """The same along the text of every attention kernel that is built."""
    tools = "/opt/rocm/llvm/bin"
    if not os.path.exists(build.LIB_PATH) or not os.path.exists(os.path.join(tools, "llvm-objdump")):
        pytest.skip("no built library, or no tools to read it with")
    lib = shutil.copy(build.LIB_PATH, tmp_path)
    subprocess.run([os.path.join(tools, "llvm-objdump"), "--offloading", lib], cwd=tmp_path, check=True, stdout=subprocess.DEVNULL)
    kernels = 0
    for image in [x for x in os.listdir(tmp_path) if x.endswith("gfx950")]:
        names = subprocess.run([os.path.join(tools, "llvm-readelf"), "-sW", image], cwd=tmp_path, check=True, capture_output=True, text=True).stdout
        names = sorted(set(re.findall(r"\s(_Z\w*16attention_kernel\w*)$", names, flags=re.M)))
        if not names:
            continue
        text = subprocess.run([os.path.join(tools, "llvm-objdump"), "-d", "--no-show-raw-insn", "--disassemble-symbols=" + ",".join(names), image],
                              cwd=tmp_path, check=True, capture_output=True, text=True).stdout
        for part in re.split(r"^(?=[0-9a-f]+ <)", text, flags=re.M)[1:]:
            kernels += 1
            for (kind, reader), states in shortest_waits(part.splitlines()).items():
                assert reader != "v_max3_f32" or states >= NEEDED[kind], (part.splitlines()[0], kind, states)
    assert kernels >= 40
