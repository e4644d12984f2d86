"""Caches whose attention is known to the key: queries of zeros weigh every key alike, and each key's values are +1 or -1
by chance, so that a column of an output is S / n, S the sum of its signs over the n keys that are seen. A key that is
lost moves every column by about 1 / n, one that comes twice or in another's place moves half of them."""


def bound(sums, number, half_step):
    """How far a kernel's output may be from sums / number. Every weight is the same power of two times 1 + e, |e| <= 2^-22
    (exp2 of an integer), its first f16 or bf16 piece that power of two, so products and their sums are whole numbers of it
    below 2^24; what e adds to the sums is off by at most 2^-24 an addition, of which there are fewer than 2^6 in a row:
    2^-18. One division, one product (2^-23) and the output's rounding follow. Where S is 0, what the second pieces leave
    when the tensor cores truncate: below 2^-22 of a product, 16 to a sum and one sum a turn, 2^-6 of a key's weight with room."""
    return abs(sums / number) * (half_step + 2.0 ** -18 + 2.0 ** -23) + 2.0 ** -6 / number
