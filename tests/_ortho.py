"""What a few steps of the orthogonalisation give in 64 bits, how far two float16 planes and float32 sums may be off from it, and
sizes that take each of its kernels.

u = 2^-24.  Held between products, a value v is off by e = 2^-23 |v| + 2^-35 (of one).  A product V = P Q of k terms is then off
by eP Q, by P eQ and by what is left out of each term, 2^-23 |p q|: of either sign in each term, so the root of the sum of their
squares; and by its sum's roundings, 3 k of up to u times what is summed so far, which is V or the root of the sum of the terms'
squares: sqrt(3 k) u of both.  That is a standard deviation at most; 3 times its norm over all of a matrix's entries is allowed
for, and 6 u of the result for the norm and the factor that X_0 is formed with, which is the same in every entry.  A product that
lost a low plane of one of its operands would be off by some 2^-12 / sqrt(3) / sqrt(2) of that norm, 1e-4."""
import torch

U = 2.0**-24


def held(v):
    return 2.0**-23 * v.abs() + 2.0**-35


def product(p, ep, q, eq):
    """(P Q, its error) of operands given with theirs."""
    v = p @ q
    square = lambda a: a.float().square()  # noqa: E731
    terms = square(p) @ square(q)
    e = (square(ep) @ square(q)).sqrt() + (square(p) @ square(eq)).sqrt() + 2.0**-23 * terms.sqrt()
    return v, e.double() + (3 * p.shape[1])**0.5 * U * (terms.sqrt().double() + v.abs())


def start(x):
    x = x.double()
    x = x / (x.norm() + 1e-7)
    return x.t().contiguous() if x.shape[0] > x.shape[1] else x


def step_of_gram(x0, order, factor):
    """(b A X, its error) for order 1, (c A^2 X, its error) for order 2."""
    t = x0.t().contiguous()
    a, ea = product(x0, held(x0), t, held(t))
    ea = ea + held(a)
    if order == 2:
        a, ea = product(a, ea, a, ea)
    p, ep = factor * a, abs(factor) * ea
    ep = ep + held(p)
    return product(p, ep, x0, held(x0))


def within(y, want, error, dtype):
    """(how far y is off, how far it may be), as norms."""
    bound = 3 * error.norm() + 6 * U * want.norm()
    if dtype is torch.float32:
        bound = bound + U * want.norm()
    else:  # its rounding, which the error moves by at most itself again
        bound = 2 * bound + (want.bfloat16().double() - want).norm()
    return (y.double() - want).norm().item(), bound.item()


# Every kernel that a product of a step can take (tests/test_ortho_tiles.py), with sides that end inside tiles and steps.
SIZES = [(70, 200), (200, 70), (300, 130), (130, 300), (100, 1217), (1448, 80), (365, 365), (410, 365), (391, 1444), (1000, 725),
         (1023, 1000), (611, 803), (803, 611), (90, 9001), (9001, 90), (1500, 3003), (3003, 1500), (1829, 1833), (2301, 1829),
         (8192, 1024), (8203, 1029), (1032, 8200), (3000, 2000), (3001, 2001), (2050, 4100), (4100, 2050), (8200, 2056),
         (4100, 4100), (3001, 8005), (8005, 3001), (5003, 5011), (5811, 4875), (9743, 9751), (11590, 9743)]
