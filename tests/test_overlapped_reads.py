"""Kernels that start under the tail of the kernel before them (programmatic dependent launch), read from their sources: what an
earlier kernel may still be writing when they start is not read through the non-coherent path, whose data has to be read-only
for as long as the kernel runs. That path is for weights, their scales and tables that no kernel of a step writes."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "deplodock_b200" / "csrc"

#: file -> what it may read through the non-coherent path: arguments of __ldg / ld_global_nc_v8, const __restrict__ pointers
READ_ONLY = {
    "emk_gemm_e4m3_sm100.cu": {"g.w_scale"},
    "emk_sdpa_kv8.cu": set(),
    "emk_kv8.cuh": set(),
    "emk_kv8_append.cu": set(),
    "emk_rmsnorm_e4m3.cu": {"w"},
    # a layer's weights, biases and rotary tables; positions, ids and cu_seqlens come from outside the step
    "emk_gemm_common.cuh": {"g.f32_bias", "g.scale", "g.residual", "g.qk_pos", "wp", "tp"},
    "emk_gemm2_sm100.cu": set(),
    "emk_gemm_chain_sm100.cu": set(),
    "emk_fmha_sm100.cu": {"cu_seqlens"},
    "emk_pointwise.cu": {"src", "table", "ids", "w", "cu_seqlens", "head", "cosb", "sinb"},
}


def non_coherent_reads(text: str) -> set[str]:
    text = re.sub(r"//[^\n]*", "", text)
    found = set()
    for m in re.finditer(r"\b(?:__ldg|ld_global_nc_v8)\(\s*(?:reinterpret_cast<[^>]*>\s*\(\s*)?\(*([A-Za-z_][\w.]*)", text):
        found.add(m.group(1))
    # a const __restrict__ parameter of a kernel: the compiler may choose the non-coherent path itself
    for kernel in re.split(r"^(?=__global__)", text, flags=re.M)[1:]:
        head = kernel[:kernel.index("{")]
        body = re.split(r"^}", kernel, flags=re.M)[0]
        if "grid_dependency_wait" in body:
            found |= set(re.findall(r"const [\w ]+\* ?__restrict__ (\w+)", head))
    return found


@pytest.mark.parametrize("name", READ_ONLY)
def test_only_weights_and_tables_are_read_as_read_only_data(name):
    assert non_coherent_reads((CSRC / name).read_text()) <= READ_ONLY[name]


def test_the_search_finds_both_kinds():
    text = """
__global__ void k(const float* __restrict__ x, const T* y, float* __restrict__ z) {
  grid_dependency_wait();
  const float a = __ldg(g.scale + i), b = __ldg(reinterpret_cast<const uint4*>(h.w + 4 * i));  // __ldg(no)
}
__global__ void ordinary(const float* __restrict__ v) {
}
"""
    assert non_coherent_reads(text) == {"g.scale", "h.w", "x"}
