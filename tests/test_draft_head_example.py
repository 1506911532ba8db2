"""The draft head's example end to end: trained, packed into 4 bits, drafting, verified."""
import runpy
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
EXAMPLE = Path(__file__).resolve().parents[1] / "examples" / "draft_head.py"


def test_trains_packs_and_drafts():
    out = runpy.run_path(str(EXAMPLE))["run"](V=8_192, Vd=2_048, K=512, rows=1_024, streams=8,
                                               steps=60, verbose=False)
    assert out["loss_last"] < 0.5 * out["loss_first"]
    assert out["bytes_packed"] < 0.3 * out["bytes_bf16"]
    # 4 bits cost little of what was learned
    assert abs(out["logprob_bf16"] - out["logprob_packed"]) < 0.1 * abs(out["loss_first"])
    assert out["accepted"]["4 bits"] >= out["accepted"]["bf16"] - 0.1
    assert out["accepted"]["bf16"] > 0.3
