"""A refusal that the library's own build has to keep: it assumes that there are no
NaNs, so a check for one must not be a comparison."""
import pytest
import torch

from locus_amd import sampler as S

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eps", [float("nan"), float("inf"), float("-inf"), 0.0])
def test_norm_eps(eps):
    s = S.Sampler(device=0, max_rows=8, max_vocab=4096, max_hist=64, max_top=4)
    x, w = torch.ones(2, 64, device="cuda"), torch.ones(64, device="cuda")
    with pytest.raises(S.SamplerError, match="eps"):
        s.add_rmsnorm_dev(x, w, {"y": torch.empty_like(x)}, eps=eps)
    s.close()
