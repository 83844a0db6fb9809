"""How far a kernel's attention may be from the exact one, from its roundings.

With p the exact probabilities, mass = sum p |v|, u half a step of the output type:
  scores      each is a float32 sum of d products, scaled: off by at most (d + 4) 2^-24 S, S the largest scaling *
              sum |q k|; a probability, the quotient of two such sums, by twice that relative error,
  exp2, sums  2^-20 covers v_exp_f32 (1 ulp) on arguments reduced by one float32 subtraction: its argument is
              off by 2^-24 of the largest score, 2 S 2^-24 log2(e) as a relative error; the sums add 2 n 2^-24,
  weights     each weight rounded by `weight` relative to itself (u of the type, or 2^-17 as a pair of bf16), fp16
              weights below 2^-14 by 2^-25 of the row's largest: n 2^-25 max |v| more,
  output      u |o| (and 2^-25 in the subnormal range of fp16).
"""
import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def bound(out, mass, score, vmax, n, d, dtype, weight):
    u = HALF[dtype]
    rel = 2 * (d + 4 + 3) * 2.0 ** -24 * score + 2.0 ** -20 + 2 * n * 2.0 ** -24
    first = (weight + rel) * mass + (n * 2.0 ** -25 * vmax if dtype == torch.float16 else 0.0)
    return first + u * (out.abs() + first) + 2.0 ** -25


def check(got, ref, vmax, n, d, dtype, weight, what=""):
    out, mass, score = ref
    tol = bound(out, mass, score, vmax, n, d, dtype, weight)
    err = (got.double().cpu() - out).abs()
    worst = float((err / tol).max()) if err.numel() else 0.0
    print(f"{what}: {worst:.3f} of the bound", flush=True)
    assert torch.isfinite(got).all() and worst <= 1.0
