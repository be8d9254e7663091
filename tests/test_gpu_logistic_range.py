"""The gates of a recurrence over the whole range of Float32 logits, open and closed, in the kernel of few steps and in that of many.

Bound.  exp(-a) is 2^t with t = -log2(e) a rounded to fp32: the constant is off by 2^-26.2 of its value and the product by 2^-24, which changes
2^t by ln 2 1.4427 |a| (2^-24 + 2^-26.2) = 0.61 |a| 2^-23 of its value.  2^t itself, the sum with 1, the reciprocal and the products behind them
are off by a few 2^-23 together: 6.  What is below 2^-126 may be taken for it or for zero: a product with such a gate is off by 2^-125."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _check(got, want, logit):
    off = (got.double() - want).abs()
    limit = (6 + 0.61 * logit.abs()) * 2.0 ** -23 * want.abs() + 2.0 ** -125
    assert bool((off <= limit).all()), f"worst {float((off / limit).max()):.3g} times its bound, at a logit of {float(logit.flatten()[(off / limit).argmax()])}"


@pytest.mark.parametrize("T", [1, 8, 9, 200])
def test_gates_keep_their_relative_error_over_their_range(T):
    import swiftrt_b200 as srt
    a = torch.cat((torch.linspace(-86, 86, 2001), torch.randn(2047) * 20, torch.tensor([0.0, -0.0, 1e-30, -1e-30, 100.0, -100.0, 300.0, -300.0]))).cuda()
    D = a.numel()
    logits = torch.full((1, T, D), 200.0, device="cuda")           # open: later steps leave the state as it is
    logits[:, 0] = a
    zero, one = torch.zeros_like(logits), torch.zeros_like(logits)
    one[:, 0] = 1.0
    s, r = torch.sigmoid(a.double()), torch.sigmoid(-a.double())
    keep = torch.ones(1, D, device="cuda")
    _check(srt.gated_recurrence(zero, logits, None, None, keep)[1][0], s, a)                 # f c
    _check(srt.gated_recurrence(one, logits)[1][0], r, a)                                    # 1 - f
    _check(srt.gated_recurrence(one, zero + 200, logits)[1][0], s, a)                        # the input gate
    hidden = srt.gated_recurrence(zero, zero + 200, None, a.expand(1, T, D).contiguous(), keep)[0]
    for t in range(T):
        _check(hidden[0, t], s, a)                                                           # the output gate


def test_slopes_of_the_gates(T=70):
    import swiftrt_b200 as srt
    a = torch.linspace(-60, 60, 4001).cuda()
    D = a.numel()
    zero = torch.zeros(1, T, D, device="cuda")
    out_grad = zero.clone()
    out_grad[:, 0] = 1.0
    logits = a.expand(1, T, D).contiguous()
    start = torch.full((1, D), 3.0, device="cuda")
    _, _, states = srt.gated_recurrence(zero, logits, None, None, start, keep=True)
    _, df, _, _, dc = srt.gated_recurrence_backward(out_grad, zero, logits, None, None, states)
    s, r = torch.sigmoid(a.double()), torch.sigmoid(-a.double())
    _check(df[0, 0], 3 * s * r, 2 * a)                              # (f and 1 - f: either may be the small one, both carry the bound)
    _check(dc[0], s, a)
