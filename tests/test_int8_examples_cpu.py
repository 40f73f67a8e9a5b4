"""The documented C++ example of a layer in 8-bit integers: it compiles against the header, and it waits for its weights before it has
them read early."""
import glob
import os
import re
import subprocess

import pytest

from conftest import ROOT

PRELUDE = """
#include "llm_infer_attn.h"
extern "C" int cudaStreamSynchronize(void*);
void example(int8_t* w8, float* w_scale, const void* w_fp16, int8_t* a8, float* a_scale, float* x, const float* last_projection,
             const float* rms, float* out, uint32_t tokens, uint32_t n_out, uint32_t k, float eps, void* stream) {
"""


def _examples():
    """The C++ blocks that have weights read early, of the documents that show how the header is used."""
    found = []
    for path in glob.glob(os.path.join(ROOT, "*.md")):
        with open(path) as f:
            text = f.read()
        if '#include "llm_infer_attn.h"' in text:
            found += [b for b in re.findall(r"```cpp\n(.*?)```", text, re.S) if "w_early = 1" in b and "attn_gemm_i8(&" in b]
    return found


def test_weights_are_waited_for_before_they_are_read_early():
    """Kernels overlap several deep, so that a product with w_early may run beside a quantisation two kernels ahead of it: between
    the kernel that writes the weights and the kernel in front of the product the host has to wait."""
    examples = _examples()
    assert examples
    for block in examples:
        code = re.sub(r"//.*|/\*.*?\*/", "", block)
        weights = re.search(r"\.w = (\w+);", code).group(1)
        writer = re.search(rf"(\w+)\.q = {weights};", code)
        if not writer:
            continue  # weights from elsewhere
        written = code.index(f"attn_quantize_i8(&{writer.group(1)}")
        calls = [m.start() for m in re.finditer(r"attn_\w+\(&", code) if m.start() > written]
        product = code.index("attn_gemm_i8(&")
        in_front = max(c for c in calls if c < product)
        assert re.search(r"cudaStreamSynchronize\(", code[written:in_front]), "the weights' writer is not waited for"


@pytest.mark.parametrize("i", range(len(_examples())))
def test_example_compiles(i, tmp_path):
    src = tmp_path / "example.cpp"
    src.write_text(PRELUDE + _examples()[i] + "}\n")
    subprocess.run(["g++", "-std=c++17", "-fsyntax-only", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src)], check=True)
