"""The Muon half of the optimiser step inside the trainers' arena."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def build():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from tests.product_runner import build_product
    return build_product


def test_a_refused_step_changes_nothing(build):
    """Coefficients that only the kernels' own check refuses (the iteration leaves its range): no AdamW half, no count, no moment."""
    import poet_amd
    r = build("tiny", 2, True, "fp32", dropout=0.0)
    A = poet_amd.Trainer(r["model"], r["crit"], lr=1e-3, weight_decay=0.1, max_norm=0.1, distributed=False, muon=dict(coeffs=(50.0, 0.0, 0.0))).arena
    A.grad.normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    before = [t.clone() for t in (A.flat, A.m, A.v, A.flat_bf16, A.flat_bf16_lo)]
    for _ in range(2):
        with pytest.raises(poet_amd.PoetHipError, match="range"):
            A.step(0.1)
    torch.cuda.synchronize()
    assert A.step_count == 0 and all(torch.equal(a, b) for a, b in zip(before, (A.flat, A.m, A.v, A.flat_bf16, A.flat_bf16_lo)))


def test_output_layers_step_by_adamw(build):
    """Learned reference points: their 2-row Linear is an output layer like the heads' last ones, so AdamW steps it (its second moment moves)."""
    import poet_amd
    r = build("tiny", 2, True, "fp32", dropout=0.0, ref_points_mode="learned", query_embedding_mode="learned")
    A = poet_amd.Trainer(r["model"], r["crit"], lr=1e-3, max_norm=0.0, distributed=False, muon=True).arena
    A.grad.normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    A.step(0.0)
    outputs = [n for n, p, _ in A.entries if p.dim() > 1 and ("reference_points" in n or ("head" in n and ".layers.2." in n) or "query_embed" in n)]
    assert "transformer.reference_points.weight" in outputs and len(outputs) >= 4
    for n, p, o in A.entries:
        owned = n in A.muon_names
        assert owned == (p.dim() > 1 and n not in outputs and "level_embed" not in n), n
        assert ((A.v[o:o + p.numel()] != 0).any().item()) != owned, n
