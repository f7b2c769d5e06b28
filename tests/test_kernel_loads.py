"""The linears, the decoders' own kernels and the exchange read what the kernel in front may have written by plain loads, as the serving and
routing kernels do (tests/test_serving_loads.py, tests/test_moe_loads.py): read-only ones may be moved above the wait for it.  Read
from the sources, since whether a compiler moves a load cannot be told from results."""
import re

import pytest

from tests.conftest import ROOT

# by file: what may be read so all the same, weights and tables that no kernel of a step writes (pointers; in __ldg)
FILES = {
    "gemv_mma.cu": (set(), {"src", "src + 1"}),   # of load_unit_values<WEIGHTS>
    "gemv_f16.cu": (set(), {"p", "q"}),           # of load_run<WEIGHTS>
    "gemm_f16.cu": ({"w_a", "w_b", "norm_w"}, {"nr + i", "nr + at"}),
    "decoder.cu": ({"w", "q_norm", "k_norm", "inv_freq"}, {"nw + lane + 32 * j"}),
    "attention_fused.cuh": (set(), {"nw + i", "nw + i + HALF"}),
    "attention_prefill.cu": (set(), set()),
    "ep.cu": ({"norm_w"}, set()),
    "moe_jobs.cuh": (set(), set()),
}


# kernels without a wait are launched behind the one in front, not beside it
WITHOUT = {"dequant.cu", "gemm_tc.cu", "gemv_f32.cu"}


def source(name):
    return re.sub(r"//[^\n]*", "", (ROOT / "joshua_b200" / "csrc" / name).read_text())


@pytest.mark.parametrize("name", FILES)
def test_what_may_be_on_its_way_is_read_by_plain_loads(name):
    text, (pointers, loads) = source(name), FILES[name]
    assert set(re.findall(r"\bconst\b[^,;(){}]*\*\s*__restrict__ (\w+)", text)) <= pointers
    assert {m for m in re.findall(r"__ldg\(((?:[^()]|\([^()]*\))*)\)", text)} <= loads
    assert "ld.global.nc" not in text


def test_the_activations_of_the_linears():
    text = source("gemv_mma.cu")
    assert len(re.findall(r"WEIGHTS \? __ldg\(src(?: \+ 1)?\) : ld_behind\(src(?: \+ 1)?\)", text)) == 2
    assert set(re.findall(r"load_unit_values<true>\((\w+)", text)) == {"norm_w", "nw"}
    text = source("gemv_f16.cu")
    assert len(re.findall(r"WEIGHTS \? __ldg\((\w)\) : ld_behind\(\1\)", text)) == 2
    assert set(re.findall(r"load_run<TYPE, true>\(([\w.]+)", text)) == {"ga.norm_w"}
    assert re.search(r"float4\* nr = reinterpret_cast<const float4\*>\(norm_w\)", source("gemm_f16.cu"))


def test_every_kernel_that_is_launched_early_is_among_them():
    from tests.test_serving_loads import SERVING

    other = {"moe.cu", "attention_chunk.cu", "attention_chunk_tiles.cu", "attention_steps.cuh", "attention_tiles.cuh", "log_probs.cu"}   # tests/test_moe_loads.py
    for path in (ROOT / "joshua_b200" / "csrc").glob("*.cu"):
        text = source(path.name)
        if path.name in WITHOUT:
            assert "launch_pdl" not in text and "ProgrammaticStreamSerialization" not in text
        elif "launch_pdl" in text or "ProgrammaticStreamSerialization" in text:
            assert path.name in {*FILES, *SERVING, *other}, path.name
