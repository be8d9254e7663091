"""The gated linear recurrence and its gradients in 64 bits, step by step, with a bound on the error of a Float32
evaluation next to every value.

The bound follows the recurrence: with gates whose relative error is at most DELTA and products and sums that each add
half a step of 2^-23, the error of the state obeys E_t <= f E_{t-1} + DELTA (|f c_{t-1}| + |i x_t| + |c_t|), whatever
the order in which spans of steps are joined (a joined span multiplies the same factors).  DELTA = 2^-20 is 16 units of
2^-24: the exponential's two units and up to ten more from the rounding of its scaled argument (|logit| <= 8), the
reciprocal's one and the products' and sums' half units."""
import torch

DELTA = 2.0 ** -20
STATE_CHUNK = 64


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """Half the spacing of the subnormal numbers: what a rounding loses at least."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def forward(update, forget, input=None, output=None, initial=None, lengths=None):
    """dict of 64-bit CPU tensors: hidden, last, states and c (all states), each with an "error" partner."""
    x, a = update.double().cpu(), forget.double().cpu()
    B, T, D = x.shape
    n = torch.full((B,), T) if lengths is None else lengths.cpu().long().clamp(0, T)
    f, nf = torch.sigmoid(a), torch.sigmoid(-a)
    i = nf if input is None else torch.sigmoid(input.double().cpu())
    o = torch.ones_like(x) if output is None else torch.sigmoid(output.double().cpu())
    c = torch.zeros(B, D, dtype=torch.float64) if initial is None else initial.double().cpu()
    e = torch.zeros_like(c)
    cs, es = [c], [e]
    for t in range(T):
        on = (t < n)[:, None]
        new = f[:, t] * c + i[:, t] * x[:, t]
        err = f[:, t] * e + DELTA * ((f[:, t] * c).abs() + (i[:, t] * x[:, t]).abs() + new.abs())
        c, e = torch.where(on, new, c), torch.where(on, err, e)
        cs.append(c)
        es.append(e)
    cs, es = torch.stack(cs, 1), torch.stack(es, 1)
    on = (torch.arange(T)[None] < n[:, None])[:, :, None]
    zero = torch.zeros_like(x)
    hidden = torch.where(on, cs[:, 1:] * o, zero)
    return {"hidden": hidden, "hidden_error": torch.where(on, es[:, 1:] * o, zero) + DELTA * hidden.abs(), "last": c, "last_error": e,
            "states": cs[:, :T:STATE_CHUNK], "states_error": es[:, :T:STATE_CHUNK], "c": cs, "c_error": es, "f": f, "nf": nf, "i": i, "o": o,
            "n": n, "on": on}


def backward(out_grad, fw, update, input=None, output=None, last_grad=None):
    """{name: (gradient, bound of the Float32 evaluation's error)} for update, forget, input, output and initial."""
    x, zero = update.double().cpu(), torch.zeros_like(update.double().cpu())
    B, T, D = x.shape
    f, nf, i, o, c, ec = fw["f"], fw["nf"], fw["i"], fw["o"], fw["c"], fw["c_error"]
    dy = torch.where(fw["on"], out_grad.double().cpu(), zero)
    x = torch.where(fw["on"], x, zero)
    g = torch.zeros(B, D, dtype=torch.float64) if last_grad is None else last_grad.double().cpu()
    e = torch.zeros_like(g)
    dc, edc = torch.zeros_like(x), torch.zeros_like(x)
    for t in range(T - 1, -1, -1):
        on = (t < fw["n"])[:, None]
        p = torch.where(on, dy[:, t] * o[:, t], torch.zeros_like(g))
        new = p + g
        err = e + DELTA * (p.abs() + g.abs() + new.abs())
        dc[:, t] = torch.where(on, new, dc[:, t])
        edc[:, t] = torch.where(on, err, edc[:, t])
        g, e = torch.where(on, new * f[:, t], g), torch.where(on, err * f[:, t], e)
    before, e_before = c[:, :-1], ec[:, :-1]
    on = fw["on"]
    live = lambda v: torch.where(on, v, zero)  # noqa: E731
    other = x if input is None else zero
    slope = f * nf
    value = live(dc * (before - other) * slope)
    size = before.abs() + other.abs()
    out = {"update": (live(dc * i), live(edc * i) + DELTA * (dc * i).abs()),
           "forget": (value, live((edc * size + dc.abs() * e_before + 4 * DELTA * dc.abs() * size) * slope)),
           "initial": (g, e + DELTA * g.abs())}
    if input is not None:
        s = torch.sigmoid(-input.double().cpu())
        out["input"] = (live(dc * x * i * s), live((edc + 4 * DELTA * dc.abs()) * x.abs() * i * s))
    if output is not None:
        s = torch.sigmoid(-output.double().cpu())
        out["output"] = (live(dy * c[:, 1:] * o * s), live(dy.abs() * (ec[:, 1:] + 4 * DELTA * c[:, 1:].abs()) * o * s))
    return out


def check(got, want, error, what=""):
    """`got` (any type) is within the evaluation's bound and one rounding of `want`, element by element."""
    got = got.cpu()
    limit = error + half_step(got.dtype) * (want.abs() + error) + smallest(got.dtype)
    off = (got.double() - want).abs()
    bad = ~(off <= limit)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values off, worst {float((off / limit).max()):.3g} times its bound"
