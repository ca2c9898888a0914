"""The prefill runtime's one pass over q and k (norms and rotations of models
with q/k norms) against the four launches it stands for."""

import os

import pytest

from kernrelay_amd import libapi, modeldir
from tests.conftest import announce

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("head_dim", [64, 128])
def test_prefill_has_the_separate_launches_bits(gpu, tmp_path, head_dim):
    announce("prefill with fused q/k norm and rotation, D=%d" % head_dim)
    cfg = dict(modeldir.PRESETS["tiny-qwen3"])
    cfg.update(num_attention_heads=6, num_key_value_heads=2, head_dim=head_dim)
    d = tmp_path / "model"
    modeldir.write_model_dir(d, cfg, seq=384, seed=5)
    fnv = set()
    for fused in ("0", "1"):
        os.environ["KR_QWEN_QK_FUSED"] = fused
        try:
            for mode in ("serial", "graph_whole", "relay_split:2"):
                r = libapi.qwen_run(d, mode, seq=384, warmup=1, iters=2)
                assert r["_rc"] == 0, r
                fnv.add(r["logits_fnv64"])
        finally:
            del os.environ["KR_QWEN_QK_FUSED"]
    assert len(fnv) == 1, fnv
