"""GPU tests of log-probabilities near 0 beside large logits
(cfops_lm_head_logprobs): the error is that of the sum of exp, not of an lse
rounded to f32."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("t", [1, 16, 20, 64, 300, 1200])  # the forward's forms
@pytest.mark.parametrize("keeps", [False, True])
def test_log_probabilities_beside_large_logits(t, keeps):
    from cpuforge_amd import ops as P
    x = torch.tensor([-3000.0, 1000.0, 1000.5, 990.25, 985.0, -7.0, 999.75], device=DEV)  # every logit exact
    head, hn = x[:, None].contiguous(), torch.ones(t, 1, device=DEV)
    tg = torch.arange(t, device=DEV) % 7
    n = P.lm_head_logprobs_keep_bytes(t, 1, 7) if keeps else 0
    keep = torch.empty(n, dtype=torch.uint8, device=DEV) if n else None
    logp, lse = torch.empty(t, device=DEV), torch.empty(t, device=DEV)
    P.lm_head_logprobs(hn, head, tg, t, 1, 7, logp, lse, P.ce_result_buffer(DEV), keep)
    want = torch.log_softmax(x.double(), 0)[tg]
    # The sum: some 32 roundings of its terms and additions, in the exponentials' arguments
    # 2^-24 of a difference of at most 16 (beyond, a term is below 2^-23 of the sum); then
    # logp's own.
    tol = 2.0 ** -24 * (want.abs() + 48)
    assert bool(((logp.double() - want).abs() <= tol).all()), (logp.double() - want).abs().max()
    exact = torch.logsumexp(x.double(), 0)
    assert bool(((lse.double() - exact).abs() <= 2.0 ** -24 * (exact.abs() + 48)).all())
