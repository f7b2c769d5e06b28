"""Prompts of routed experts behind one another: the lists of one must not be those of the one before."""
import pytest

from tests.test_gpu_paged_decoder import ids

pytestmark = pytest.mark.gpu


def test_a_prompt_behind_a_longer_one():
    import torch

    from joshua_b200.moe_decoder import MoeDecoderConfig
    from joshua_b200.paged import PagedMoeDecoder

    cfg = MoeDecoderConfig(layers=2, hidden=1024, q_heads=8, kv_heads=2, head_dim=128, n_expert=8, n_used=2, moe_inter=256, vocab=2048)

    def decoder():
        return PagedMoeDecoder(cfg, torch.device("cuda", 0), batch=2, max_ctx=320, kv_type="q8_0", seed=1)

    alone = decoder()
    alone.prefill(ids(33, 2), sequence=1)
    for _ in range(40):
        dec = decoder()
        dec.prefill(ids(40, 1), sequence=0)
        dec.prefill(ids(33, 2), sequence=1)
        assert bool((dec.logits[1] == alone.logits[1]).all())
