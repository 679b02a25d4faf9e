"""How far the attention over a 4-bit context is off as a whole, next to the worst case a value (_context_mx_checks).

The kernel rounds three times: the query, scaled, to 8 significant bits (``q (1 + x)`` a channel), the
probabilities to bf16 (``p (1 + y)`` a position and query row, the sum taken of the rounded ones) and the result to
bf16 (``o (1 + z)`` a value), each by at most 2^-8. To first order the result ``o = sum p v / sum p`` is then
off by

    sum_j p_j (y_j + s sum_c q_c k_jc x_c) (v_j - o) / sum p + z o

for a softmax scale ``s``. The roundings are independent of each other and of the values, so that the squares add
up: with ``t_j^2 = s^2 sum_c q_c^2 k_jc^2`` the error's norm over a request's rows of a head is near that of

    e = r sqrt(o^2 + sum_j p_j^2 (1 + t_j^2) (v_j - o)^2),    p normalized

where ``r`` is a rounding's root mean square, 2^-8 / sqrt(3) at the foot of a binade and 0.74 of that over one.
``check_norm`` asks for at most ``e`` with r = 2^-8, the largest rounding in the place of the mean one: 1.7 to 2.3
times what is expected, and less than a fault of 1 or 2 in a hundred makes. Sums in float32 (2^-24 times the root
of some thousand terms) and the matrix instruction's cut of small products (2^-13 of a group's largest, where the
query's rounding takes 2^-8 of each) are far below either.
"""

import torch


def attention(query: torch.Tensor, rows, lens_q, scale: float):
    """Per request the result ``(tokens, hq, d)`` in float64 and ``e / r (hq,)``, over its tokens and channels."""
    at, d = 0, query.shape[-1]
    for kv, n in zip(rows, lens_q):
        q = query[at:at + n].double()
        at += n
        group = q.shape[1] // kv.shape[1]
        results, norms = [], []
        for h in range(kv.shape[1]):
            k, v = kv[:, h, :d].double(), kv[:, h, d:].double()
            x = q[:, h * group:(h + 1) * group].reshape(-1, d)
            p = torch.softmax(x @ k.T.contiguous() * scale, -1)
            o = p @ v
            w = p.square() * (1 + scale ** 2 * (x.square() @ k.square().T.contiguous()))
            # sum_d sum_j w_j (v_j - o)^2
            spread = (w @ v.square()).sum(-1) - 2 * (o * (w @ v)).sum(-1) + o.square().sum(-1) * w.sum(-1)
            results.append(o.view(n, group, d))
            norms.append((o.square().sum(-1) + spread.clamp(min=0)).view(n, group).sum(0).sqrt())
        yield torch.cat(results, 1), torch.cat(norms)


def check_norm(out: torch.Tensor, query: torch.Tensor, rows, lens_q, scale: float) -> float:
    """``out`` and ``query (tokens, hq, d)`` (what attends: normed and rotated) against float64, ``rows`` the contexts
    ``(positions, hkv, 2 d)``; returns the largest error of a request's head in units of its bound."""
    at, worst = 0, 0.0
    for b, (kv, n) in enumerate(zip(rows, lens_q)):
        got = out[at:at + n].double()
        if kv.shape[0] == 0 or n == 0:
            assert (got == 0).all(), f"request {b}: no context, but not zeros"
        else:
            want, e = next(attention(query[at:at + n], [kv], [n], scale))
            off = (got - want).square().sum((0, 2)).sqrt() / (2.0 ** -8 * e)
            assert (off <= 1).all(), (f"request {b} ({kv.shape[0]} positions), head {int(off.argmax())}: off by "
                                      f"{off.max():.2f} times its bound")
            worst = max(worst, float(off.max()))
        at += n
    return worst
