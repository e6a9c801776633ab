"""How many digits the adapters' delta has, by norms over many elements: a bound that a lost half of x.A^T exceeds.

With y_add = 0 the result is round(delta + e).  Its error's norm is the rounding's, I = |round(delta) - delta|,
where e is small beside a step, and at most about I + |e|.  e has two parts:
* x.A^T as hi + lo, eps^2 of it: nothing beside I (2^-16 and 2^-22 against 2^-9.2 and 2^-12.2 on average);
* fp32 sums that a tensor core rounds towards zero once per sixteen products: the running sum loses half a last digit
  (2^-24 to 2^-25 of it, 0.36 x 2^-23 on average over a binade) each time, always inwards.  Of products of random sign
  it is two thirds of the last sum on average, which makes 0.24 x 2^-23 x K / 16 of x.A^T, and as much of delta.
I's own spread over n elements is 1 / sqrt(2 n) of it or so; 3% are allowed.
One number of 16 bits for x.A^T adds an error as large as I (independent of it): sqrt(2) I."""
import torch


def rounding(delta, dtype):
    """The norm of the error that the result's own rounding makes."""
    return (delta.to(dtype).double() - delta).norm().item()


def bound(delta, k, dtype):
    return 1.03 * rounding(delta, dtype) + 0.25 * 2.0 ** -23 * (k / 16) * delta.norm().item()


def parts(t, dtype, numbers):
    """t [.., R] in 64 bits as a sum of `numbers` numbers of dtype."""
    out = torch.zeros_like(t)
    for _ in range(numbers):
        out += (t - out).to(dtype).double()
    return out
