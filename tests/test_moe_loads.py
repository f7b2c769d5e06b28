"""Kernels that are launched while the one in front still runs wait for it in their first statements.  Read-only loads may be moved above
that wait, so what the kernel in front may have written is read by plain loads.  Read from the sources, as for the serving kernels
(tests/test_serving_loads.py), since whether a compiler moves a load cannot be told from results."""
import re

from tests.conftest import ROOT

WEIGHTS = {"router", "bias", "norm_w"}


def source(name):
    return re.sub(r"//[^\n]*", "", (ROOT / "joshua_b200" / "csrc" / name).read_text())


def test_routing_and_lists():
    text = source("moe.cu")
    assert set(re.findall(r"\bconst \w+\*\s*__restrict__ (\w+)", text)) <= WEIGHTS
    for load in re.findall(r"__ldg\(([^;]*);", text):
        assert re.match(r"(b\[q\] \+ j|b \+ j|g \+ j)\)", load), load   # router rows and norm weights


def test_the_split_of_activations():
    text = source("gemm_f16.cu")
    kernel = text[text.index("split_f16_kernel("):]
    kernel = kernel[:kernel.index("\n}\n")]
    assert set(re.findall(r"\bconst \w+\*\s*__restrict__ (\w+)", kernel)) <= WEIGHTS
    assert not re.search(r"__ldg\(xr", kernel)


def test_chunks_and_scores():
    for name in ("attention_chunk.cu", "attention_chunk_tiles.cu", "attention_steps.cuh", "attention_tiles.cuh", "log_probs.cu"):
        text = source(name)
        assert not re.search(r"\bconst\b[^,;(){}]*\*\s*__restrict__", text)
        for load in re.findall(r"__ldg\(([^;]*);", text):
            assert not re.search(r"\b(src|x|qkv|logits|len|first|token)\b|table\b", load), load
