"""Tensors with a tangent of torch's forward mode: there is no derivative for them, so the key-value cache and beam search's selection refuse them, as they refuse tensors that require gradients."""
import pytest


def _dual(x):
    import torch
    return torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))


def test_what_wants_gradients():
    """(no device)"""
    import torch
    from bam_amd.host import BamError, _wants_gradients
    from bam_amd.kv import KVCache
    x, y = torch.ones(2, 3), torch.ones(2, 3, requires_grad=True)
    assert not _wants_gradients(x) and _wants_gradients(y)
    with torch.autograd.forward_ad.dual_level():
        z = _dual(x)
        assert not _wants_gradients(x) and _wants_gradients(z) and _wants_gradients(z[:1])
        with torch.no_grad():                        # torch carries tangents on here too
            assert not _wants_gradients(y) and _wants_gradients(z)
        with pytest.raises(BamError, match="tangent"):
            KVCache._no_grad(None, z, "k")
        KVCache._no_grad(None, x, "k")
        KVCache._no_grad(None, torch.autograd.forward_ad.unpack_dual(z).primal, "k")


@pytest.mark.gpu
def test_refused_by_each_call():
    import torch
    import bam_amd
    from test_gpu_kv import Cache, _i32
    with Cache(bam_amd, 8, 1, 64, "bf16") as c, torch.autograd.forward_ad.dual_level():
        x, lens, table = torch.ones(1, 1, 64, dtype=c.dtype, device="cuda"), _i32([1]), torch.zeros(1, 1, dtype=torch.int32, device="cuda")
        w, angle = x[0, 0].clone(), torch.ones(1, 32, device="cuda")
        logits, scores = torch.ones(2, 9, device="cuda"), torch.zeros(1, 2, device="cuda")
        calls = [(c.kv.append, [x, x.clone(), lens, table], {"q": x.clone(), "q_norm": w, "k_norm": w.clone(), "cos": angle, "sin": angle.clone()}), (c.kv.attend, [x.clone(), lens, table], {}),
                 (bam_amd.beam_select, [logits, scores], {})]
        for call, args, kw in calls:
            call(*args, **kw)
            for i, a in enumerate(args):
                if a.dtype.is_floating_point:
                    with pytest.raises(bam_amd.BamError):
                        call(*args[:i], _dual(a), *args[i + 1:], **kw)
            for name in kw:
                with pytest.raises(bam_amd.BamError):
                    call(*args, **{**kw, name: _dual(kw[name])})
