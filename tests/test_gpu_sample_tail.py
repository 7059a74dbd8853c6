"""The lightest weight that plamo_kernel_sample draws.  Weights are whole multiples of 2^-S of the largest, S = 46 up to
n = 2^17 - 1 and one less for each doubling from 2^17 on, so that one above 2^-(S + 1) counts and one below does not.  A
uniform number of 1 takes the last token that counts."""
import math

import pytest
import torch

from paged_common import sample

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,least", [(5, 47), (1 << 15, 47), ((1 << 17) - 1, 47), (1 << 17, 46), ((1 << 18) - 1, 46),
                                     (1 << 18, 45), (1 << 19, 44), ((1 << 20) - 1, 44), (1 << 20, 43)])
def test_the_lightest_token(n, least):
    # a fifth of a factor of two on either side: FP32 holds the logit to 2^-19
    logits = torch.full((2, n), -math.inf, device="cuda")
    logits[:, 2] = 3.0
    logits[0, n - 1] = 3.0 - (least - 0.2) * math.log(2)
    logits[1, n - 1] = 3.0 - (least + 0.2) * math.log(2)
    token, prob = sample(logits, n, torch.ones(2, device="cuda"))
    assert token.tolist() == [n - 1, 2, -7]
    assert abs(prob[0].item() / 2.0 ** (1 - least) - 1) < 1e-6 and prob[1].item() == 1
