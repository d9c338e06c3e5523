"""The example that serves from a key-value cache: in 8 bits, and as a beam search, over caches of which a part is resident."""
import pytest

from test_gpu_parity import bam  # noqa: F401  (the module fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("resident", [1.0, 0.4])
def test_eight_bits(bam, resident):
    """layers with and without a window, prompts and then tokens, against plain torch over the keys and values that the cache has: an output is off by the rounding of what it is made of, a few
    2^-8 of the largest (2^-5 is allowed, a missing token or page is off by more)"""
    from bam_amd.examples import kv_serve
    got = kv_serve.main(["--batch", "5", "--prompt", "300", "--steps", "6", "--layers", "3", "--resident", str(resident), "--eight", "--check"])
    assert not got["aborted"] and got["worst"] < 2.0 ** -5, got
    assert (got["page_reads"] > 0) == (resident < 1), got


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("resident", [1.0, 0.5])
@pytest.mark.parametrize("beams,steps", [(4, 20), (1, 3), (3, 40)])
def test_beams(bam, eight, resident, beams, steps):
    """each step's choice against the definition in 64 bits; each beam's layers against plain torch over its own tokens, wherever its parents' blocks went; the sums of the beams that are left add up"""
    import torch
    from bam_amd.examples import kv_serve
    from test_gpu_beam import _check
    got = kv_serve.main(["--batch", "3", "--prompt", "150", "--steps", str(steps), "--layers", "2", "--resident", str(resident), "--beams", str(beams), "--check"] + (["--eight"] if eight else []))
    assert not got["aborted"] and got["worst"] < 2.0 ** -5, got
    assert got["tokens"].shape == (3, beams, steps) and len(got["logs"]) == steps
    sums = torch.zeros(3 * beams, dtype=torch.float64)
    for k, (logits, before, parents, tokens) in enumerate(got["logs"]):
        after = got["logs"][k + 1][1] if k + 1 < steps else got["sums"]
        _check((after, parents.view(3, beams), tokens.view(3, beams)), logits, before, beams)
        p, t = parents.cpu().long(), tokens.cpu().long()
        sums = sums[p] + torch.log_softmax(logits.cpu().double(), 1)[p, t]
    # roundings of a sum at each step, and what a step's logarithm is off by
    assert bool(((got["sums"].cpu().double().flatten() - sums).abs() <= steps * (2.0 ** -19 + 1.01 * 2.0 ** -24 * sums.abs())).all())
