"""How exact decode over a small cache has to be, from the sizes of its own terms.

fp32 outputs.  The kernels take the sums that a plain fp32 evaluation takes, in another order, and
hold queries, probabilities, their products with a scale, and the middles of K's and V's groups as
two fp16 halves: 22 bits, each off by at most 2^-22 of itself, one independent of the other.  Against
24 bits that is four times a plain evaluation's error in the scores; and three such factors in each
term of the output leave 2^-22 (as a root mean square) of sqrt(sum_t p_t^2 u_t^2), u = |s (n - 8)| +
|z + 8 s|, to be doubled for what a tensor core's sums drop.  So, as root mean squares over the outputs,
err <= 4 err(fp32) + 2^-21 terms.

16-bit outputs.  The rounding of the output must be nearly all of the error: with N tokens of
scores of unit spread, probabilities and their products in fp16 (three roundings of 2^-11) leave
sqrt(e / N) 2^-11 of the terms, under a fifth of a bf16 output's own rounding from N = 300 on, and
0.2 in the square is 2 % in the sum:  err <= 1.1 err(rounding).

Weights are fp32 whatever the outputs: relative to each,  err <= 4 err(fp32) + 2^-20 (exp2 and the
sums), and with 16-bit queries over 4 bits 2^-19 Q more for subnormal nibbles, Q = max_t
sum_d |q_d s n_d| / sqrt(D)."""

import torch


def attention(q, k, v, dtype, p_bits=None):
    """Decode attention of q [B, Hq, D] over k, v [B, Hkv, N, D] and the summed probabilities, every
    step in ``dtype``; p_bits: the probabilities rounded to that many bits (a planted loss)."""
    b, hq, d = q.shape
    qs = q.to(dtype).view(b, k.size(1), -1, d)
    k, v = k.to(dtype), v.to(dtype)
    p = torch.softmax(qs @ k.transpose(2, 3) / torch.tensor(d, dtype=dtype).sqrt(), -1)
    if p_bits:
        m, e = torch.frexp(p)
        p = torch.ldexp((m * 2 ** p_bits).round() / 2 ** p_bits, e)
    return (p @ v).reshape(b, hq, d), p.sum(2)


def terms(q, k, parts):
    """sqrt(sum_t p_t^2 u_t^2): u = |s (n - 8)| + |z + 8 s|, or |v| of a plain cache."""
    b, hq, d = q.shape
    p = torch.softmax(q.double().view(b, k.size(1), -1, d) @ k.double().transpose(2, 3) / d ** 0.5, -1)
    return (p.square() @ parts.double().square()).sqrt().reshape(b, hq, d)


def int4_parts(values, scales):
    """|s (n - 8)| + |z + 8 s| and |s n| of dequantised values [..., D]."""
    s, z = (x.double().repeat_interleave(32, -1) for x in scales.double().unbind(-2))
    return (values - z - 8 * s).abs() + (z + 8 * s).abs(), (values - z).abs()


def rms(x):
    return x.double().square().mean().sqrt().item()


def output_limit(dtype, want, plain32, size):
    if dtype == torch.float32:
        return 4 * rms(plain32.double() - want) + 2.0 ** -21 * rms(size)
    return 1.1 * rms(want.to(dtype).double() - want)


def weight_limit(dtype, want, plain32, q, nibbles=None):
    limit = 4 * rms(plain32.double() / want - 1) + 2.0 ** -20
    if nibbles is not None and dtype != torch.float32:
        group = q.size(1) // nibbles.size(1)
        big = nibbles.repeat_interleave(group, 1) @ q.double().abs()[..., None]
        limit += 2.0 ** -19 * (big.max() / q.size(2) ** 0.5).item()
    return limit
