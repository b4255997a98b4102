"""Cache attention from its definition in 64 bits, by torch on the tensors'
device, and the error that the documented arithmetic may make: test
infrastructure only.  For single sequences and chosen rows, so that long ones
stay cheap."""
import torch


def attention64(q, k, v, positions, scale, window=0, absent=None):
    """q [rows][heads][dim] at `positions` over the tokens k, v
    [length][kv_heads][dim] (bf16 or wider), but for the tokens that `absent`
    [length] marks.  Returns out, its bound, lse, its bound, all float64; with
    them the weights [rows][heads][length] and their bound.

    The bound: products of bf16 are exact and their f32 sums within 2^-20 of
    the sum of magnitudes; a weight enters the product with V in f16, with a
    relative error of 2^-11 and, below 2^-25 of the row's largest, an absolute
    one of 2^-36 of that; powers, sums and quotients in f32 within 2^-17; the
    result is rounded to bf16 (2^-8)."""
    q, k, v = q.double(), k.double(), v.double()
    rows, heads, _ = q.shape
    group = heads // k.shape[1]
    pos = torch.as_tensor(positions, device=q.device)[:, None]
    tok = torch.arange(k.shape[0], device=q.device)
    sees = tok <= pos
    if window:
        sees &= tok > pos - window
    if absent is not None:
        sees &= ~absent
    got = []
    for h in range(heads):
        kh, vh, x = k[:, h // group], v[:, h // group], q[:, h]
        s = torch.where(sees, scale * (x @ kh.T), -torch.inf)
        eps = (torch.where(sees, x.abs() @ kh.abs().T, 0.).amax(1) * abs(scale) * 2.0 ** -20)
        lse = torch.logsumexp(s, 1)
        p = torch.where(sees, torch.exp(s - lse[:, None]), 0.).nan_to_num(0.)
        out, size = p @ vh, p @ vh.abs()
        part = (2.0 ** -11 + 2.0 ** -17 + 2 * eps)[:, None] * size + \
            2.0 ** -36 * p.amax(1)[:, None] * (sees.double() @ vh.abs())
        got.append((out, part + 2.0 ** -8 * (out.abs() + part), lse,
                    eps + 2.0 ** -20 * lse.abs().clamp(min=1).nan_to_num(posinf=1),
                    p, p * (2 * eps + 2.0 ** -17)[:, None]))
    return tuple(torch.stack(t, 1) for t in zip(*got))


def within(got, ref, tol, what):
    over = (got.double() - ref).abs() - tol
    same = torch.isinf(ref) & (got.double() == ref)
    over = torch.where(same, -1., over)
    assert not over.isnan().any(), what
    worst = float(over.max()) if over.numel() else 0.0
    assert worst <= 0, f"{what}: {worst} over the bound"
