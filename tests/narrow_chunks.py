"""The tolerance of chunks of few rows, whose probabilities are not rounded to bf16 but kept in two bf16 parts, for the tests.

The first part is a probability cut off after its first 8 bits, so that less than 2^-7 of the power of two below it is left, and the
second is that rest rounded: by half a step of at most 2^-15 of that power, so by 2^-16 of the probability. attend_reference
allows 1.01 · 2^-8 of A = Σ p|v| / Σ p for this rounding; here 1.01 · 2^-16 of it takes that place."""
from attend_reference import U, attended


def attended_narrow(q, k, v, first, **options):
    """attend_reference's outputs, and the tolerance for probabilities of two parts."""
    want, tol = attended(q, k, v, first, **options)
    a, _ = attended(q, k, v.abs(), first, **options)
    return want, tol - 1.01 * (U - 2.0 ** -16) * a
