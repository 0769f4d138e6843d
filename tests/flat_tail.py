"""Rows of one token of weight 1 and a flat tail of tiny ones, whose sums have a closed form."""
import math
from fractions import Fraction

import numpy as np


def rows(vocab, distance, top_ps, us):
    """(logits, params, u, wanted rank in the tail or -1 for the top token, wanted share) of one row per top_p and u, T = 1."""
    logits = np.full(vocab, 4 - distance, np.float32)
    top = vocab // 3
    logits[top] = 4
    w = Fraction(math.exp(float(logits[0]) - 4.0))
    out = []
    for tp in top_ps:
        total = 1 + (vocab - 1) * w
        tail = vocab - 1
        if np.float32(tp) < 1:
            tail = min(tail, max(0, math.ceil((Fraction(float(np.float32(tp))) * total - 1) / w)))
        kept = 1 + tail * w
        for u in us:
            target = Fraction(float(np.float32(u))) * kept
            rank = -1 if target < 1 else math.floor((target - 1) / w)
            out.append(((1.0, tp, 0, 0.0), u, rank, float((1 if rank < 0 else w) / kept)))
    return logits, top, float(w), out


def check(run, vocab, distance):
    """run(logits, params, u) -> (tokens, probs). A token's weight is off by half of the least part that vocab leaves it (one word up
    to 2^17 tokens, which takes vocab weights of 1 below 2^62, then a second one, which takes a count and further parts of as
    many), or by 2^-52 of itself (the exponential's last bits), so a sum up to the drawn token, and the one up to top_p's last, by
    that per token and by 2^-51 where they are compared: in ranks, these over the weight, and one for the floor."""
    us = [1 - 2.0 ** -24, 1 - 2.0 ** -21, 1 - 2.0 ** -19, 0.99999, 1 - 1e-6, 0.5]
    logits, top, w, want = rows(vocab, distance, [1.0, 0.99999, 1 - 2.0 ** -20], us)
    tokens, probs = run(np.tile(logits, (len(us), 1)), want, us)
    bits, count_bits = 62 - (vocab - 1).bit_length(), vocab.bit_length()
    part = 2.0 ** -(min(bits, 51) + (0 if vocab <= 1 << 17 else min(40, 64 - count_bits - (vocab - 1).bit_length())))
    slack = 2 * ((vocab * (part / 2 + 2.0 ** -52 * w) + 2.0 ** -51) / w) + 1
    seen = 0
    for (params, u, rank, share), t, p in zip(want, tokens, probs):
        got = -1 if t == top else int(t) - (t > top)
        assert abs(got - rank) <= slack if rank >= 0 else got == -1, (params, u, rank, got, slack)
        assert abs(p - share) <= 2.0 ** -23 * share, (params, u, share, p)
        seen += rank >= 0
    assert seen >= 4
