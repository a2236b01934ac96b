"""CPU: what a SelectionStep with attention says of itself (buffers and accounting
need no GPU)."""
import importlib

import pytest
import torch

P = importlib.import_module("10_20_b200.pipeline")
S = importlib.import_module("10_20_b200.synth")
LENS = [4097, 9000, 700]


@pytest.fixture(scope="module")
def case():
    return S.make_query_case(3, 64, LENS, P=256, take=12, window=64, topk=2048, seed=3, device="cpu", latent_dim=576)


def test_bytes_of_a_step_with_attention(case):
    q = torch.zeros((3, 24, 576), dtype=torch.bfloat16)
    plain = P.SelectionStep(case, gather=False).algorithmic_bytes()
    step = P.SelectionStep(case, gather=False, attention=(q, 0.07)).algorithmic_bytes()
    assert "attend" not in plain
    # attended rows: 12 pages and the 64 + 64 tokens of sink and tail; 12 pages, the sink and the 808 tokens behind the
    # last whole bucket; all 700
    rows = 12 * 64 + 128, 12 * 64 + 64 + 9000 - 8192, 700
    want = sum(rows) * 576 * 2 + 3 * 24 * ((576 + 512) * 2 + 4)
    assert step["attend"] == want
    assert step["total"] == plain["total"] + want
    assert {k: v for k, v in step.items() if k not in ("attend", "total")} == {k: v for k, v in plain.items() if k != "total"}


@pytest.mark.parametrize("q,scale,word", [
    (torch.zeros((2, 24, 576), dtype=torch.bfloat16), 0.07, "query row"),
    (torch.zeros((3, 24, 512), dtype=torch.bfloat16), 0.07, "pool"),
    (torch.zeros((3, 24, 576), dtype=torch.float16), 0.07, "pool"),
    (torch.zeros((3, 24, 576)), 0.07, "bfloat16"),
    (torch.zeros((3, 576), dtype=torch.bfloat16), 0.07, "rows, heads"),
    (torch.zeros((3, 1025, 576), dtype=torch.bfloat16), 0.07, "heads"),
    (torch.zeros((3, 24, 577), dtype=torch.bfloat16)[..., 1:], 0.07, "16-byte"),
    (torch.zeros((3, 24, 576), dtype=torch.bfloat16), float("inf"), "finite"),
])
def test_step_refuses_queries_when_made(case, q, scale, word):
    with pytest.raises(ValueError, match=word):
        P.SelectionStep(case, gather=False, attention=(q, scale))


def test_step_refuses_a_latent_pool_of_another_width():
    narrow = S.make_query_case(1, 64, [700], P=256, take=12, window=64, topk=2048, seed=3, device="cpu", latent_dim=320)
    with pytest.raises(ValueError, match="latent"):
        P.SelectionStep(narrow, gather=False, attention=(torch.zeros((1, 4, 320), dtype=torch.bfloat16), 0.07))
