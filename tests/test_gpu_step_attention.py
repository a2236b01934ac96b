"""GPU: SelectionStep(attention=) in the operator-by-operator modes, eager and captured."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu

P = importlib.import_module("10_20_b200.pipeline")
S = importlib.import_module("10_20_b200.synth")
L = importlib.import_module("10_20_b200.latent_attention")


@pytest.mark.parametrize("kw,selection", [(dict(fused=False), 5), (dict(fused=False, fused_route_pages=False), 5),
                                          (dict(ratio=(1, 3)), 2), (dict(gather=True), 3)])
def test_modes(cuda_dev, kw, selection):
    case = S.make_query_case(4, 64, [4097, 9000, 700, 20000], P=512, take=12, window=64, topk=2048, seed=5,
                             device="cuda:0", latent_dim=576)
    q = torch.randn((4, 24, 576), generator=torch.Generator(device="cuda:0").manual_seed(1), device="cuda:0")
    q = q.to(torch.bfloat16)
    step = P.SelectionStep(case, **{"gather": False, **kw}, attention=(q, 0.07))
    step.run()
    torch.cuda.synchronize()
    want = [t.clone() for t in L.attend_slots(q, case.latent, None, step.physical, 0.07)]
    assert all(torch.equal(x, y) for x, y in zip(step.attended, want))
    if "ratio" not in kw:
        other = P.SelectionStep(case, gather=False, attention=(q, 0.07))
        other.run()
        assert all(torch.equal(x, y) for x, y in zip(other.attended, want))
        live = (step.physical >= 0).sum(1).tolist()      # the rows that algorithmic_bytes counts, or fewer
        row = step.algorithmic_bytes()["attend"] - 4 * 24 * ((576 + 512) * 2 + 4)
        assert sum(live) * 1152 <= row
    step.capture()
    for t in step.attended:
        t.zero_()
    step.replay()
    assert all(torch.equal(x, y) for x, y in zip(step.attended, want))
    assert step.launches() >= selection + 1
