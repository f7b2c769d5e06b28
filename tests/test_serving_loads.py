"""Kernels that are launched while the one in front still runs wait for it in their first statements.  Read-only loads (`__ldg`, or plain ones
through `const __restrict__`) may be moved above that wait, so what the kernel in front may have written is read by plain loads: activations,
positions, lengths, page tables, logits.  Read from the sources, since whether a compiler moves a load cannot be told from results."""
import re

import pytest

from tests.conftest import ROOT

SERVING = ["rope.cu", "rope.cuh", "kv_cache.cu", "kv_pages.cuh", "attention_paged.cu", "attention_paged.cuh", "attention_lead.cu", "sample.cu"]


@pytest.mark.parametrize("name", SERVING)
def test_nothing_that_may_be_on_its_way_is_read_only(name):
    text = re.sub(r"//[^\n]*", "", (ROOT / "joshua_b200" / "csrc" / name).read_text())
    assert not re.search(r"\bconst\b[^,;(){}]*\*\s*__restrict__", text)
    for load in re.findall(r"__ldg\(([^;]*);", text):
        assert not re.search(r"\b(src|x|qkv|logits|len|seq)\b|table\b|\ba\.pos\b", load), load
