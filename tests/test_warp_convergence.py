"""CPU test of a rule in the CUDA sources: tensor-memory loads and stores are .sync.aligned.

Every lane of the warp has to execute such an instruction together. Where lanes part before it (one lane signals a barrier,
rows past the matrix skip their store) nothing but a __syncwarp() promises that they have met again, so each helper that
issues one begins with it.
"""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "lynnreal_omni_b200" / "csrc"
HELPER = re.compile(r"__device__ __forceinline__ void (\w+)\([^{;]*\) \{(.*?)\n?\}\n", re.S)


def helpers(text):
    """Bodies of the helpers that hold a tensor-memory load or store."""
    for name, body in HELPER.findall(text):
        if re.search(r"tcgen05\.(ld|st)\.sync\.aligned", body):
            yield name, body


@pytest.mark.parametrize("source", ["lr_tc.cuh", "lr_attention_packed.cu", "lr_gemm_sm100.cu", "lr_attention.cu"])
def test_tensor_memory_accesses_begin_with_a_converged_warp(source):
    text = (CSRC / source).read_text()
    found = list(helpers(text))
    assert len(found) == len(re.findall(r"tcgen05\.(?:ld|st)\.sync\.aligned", text)) >= 1
    assert [name for name, body in found if not body.lstrip().startswith("__syncwarp();")] == []
