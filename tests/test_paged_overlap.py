"""CPU: whether rows of an output meet rows of an input, against sets of bytes."""
import ctypes as C
import random

from pet_b200 import lib as L


def meets(a, b, tokens):
    def covered(r):
        at, tok, head, heads, size = r
        return {at + t * tok + h * head + i for t in range(tokens) for h in range(heads) for i in range(size)}
    return bool(covered(a) & covered(b))


def test_rows_overlap_where_they_share_a_byte():
    fn = L.load().petb200_debug_rows_overlap
    fn.argtypes, fn.restype = [C.POINTER(C.c_longlong), C.POINTER(C.c_longlong), C.c_int], C.c_int
    rng = random.Random(7)
    found = [0, 0]
    for _ in range(20000):
        tokens = rng.choice([1, 1, 2, 3, 7])
        tok = rng.choice([0, 6, 24, 25, -24, 40])
        rows = []
        for _ in range(2):
            size, heads = rng.choice([2, 4]), rng.choice([1, 2, 5])
            head = rng.choice([0, size, size + 1, 8, 60, 100, -5])
            rows.append((1000 + rng.randrange(-90, 90), tok, head, heads, size))
        got = fn((C.c_longlong * 5)(*rows[0]), (C.c_longlong * 5)(*rows[1]), tokens)
        assert bool(got) == meets(*rows, tokens), (rows, tokens)
        found[got] += 1
    assert min(found) > 2000
    # other token strides: told apart where the ranges do not meet, refused where they do
    a, b = (1000, 64, 8, 2, 8), (1000 + 4 * 64, 32, 8, 2, 8)
    assert not fn((C.c_longlong * 5)(*a), (C.c_longlong * 5)(*b), 4)
    assert fn((C.c_longlong * 5)(*a), (C.c_longlong * 5)(1016, 32, 8, 2, 8), 4)
