"""Calls of linear attention that reach every shape of its walk over the chunks (state rows, columns a workgroup, sequences split or not), among them
those that only much work takes. Large ones repeat a few heads' data over heads and sequences: all the repetitions give the same bits.

A case: types, sequences (their number and length, or packed lengths), the data's heads and shared heads, how often the sequences and the heads are
repeated, dim, value_dim, whether there is a backward pass."""
F32, F16, BF16 = 0, 1, 2
ALL, SIXTEEN = (F32, F16, BF16), (F16, BF16)


def case(types, lengths, heads, kv_heads, dim, value_dim, sequences=1, copies=1, packed=False, train=True):
    return dict(types=types, lengths=list(lengths), heads=heads, kv_heads=kv_heads, dim=dim, value_dim=value_dim, sequences=sequences, copies=copies, packed=packed,
                train=train)


CASES = (
    # Every width of the state and of a workgroup, whole and partial, a last chunk of any length, shared heads; and split sequences of the same.
    [case(ALL, [n], 4, kv, dim, dv, sequences=2) for n, kv, dim, dv in (
        (150, 2, 32, 16), (129, 4, 30, 13), (150, 2, 32, 32), (70, 1, 64, 16), (101, 4, 49, 31), (150, 2, 32, 64), (90, 4, 17, 37), (150, 2, 64, 64), (150, 4, 128, 64),
        (77, 2, 111, 50), (130, 2, 256, 64), (150, 2, 128, 128), (100, 4, 101, 83), (130, 2, 256, 128), (97, 2, 250, 253), (64, 2, 128, 128), (30, 2, 60, 100), (31, 4, 128, 128),
        (150, 2, 30, 100))]
    + [case(ALL, [n], 2, kv, dim, dv) for n, kv, dim, dv in (
        (2111, 1, 32, 16), (2000, 2, 20, 30), (2111, 1, 64, 16), (2049, 2, 40, 32), (2111, 1, 32, 64), (2111, 1, 64, 64), (2111, 1, 128, 128), (2200, 2, 97, 70), (2111, 1, 256, 256),
        (2111, 2, 256, 200), (2111, 2, 200, 64), (2111, 1, 128, 256), (2111, 1, 29, 99),
        (2111, 1, 128, 64))]
    # 128 columns and two workgroups a CU: enough work that the estimate takes them. Forwards,
    + [case((BF16,), [700], 2, 1, dim, dv, sequences=16, copies=16, train=False) for dim, dv in ((32, 128), (64, 101), (128, 128), (101, 77))]
    + [case((F32,), [300], 2, 1, dim, dv, sequences=16, copies=16, train=False) for dim, dv in ((32, 128), (64, 101))]
    # with gradients,
    + [case((BF16,), [700], 2, kv, 128, 128, sequences=33, copies=2) for kv in (1, 2)]
    + [case((BF16,), [700], 2, kv, dim, dv, sequences=16, copies=8) for kv, dim, dv in ((2, 128, 60), (1, 77, 101), (1, 101, 32))]
    + [case((F32,), [300], 2, kv, dim, dv, sequences=16, copies=8) for kv, dim, dv in ((1, 128, 60), (2, 101, 32))]
    # split,
    + [case((BF16,), [6000], 2, 1, dim, dv, sequences=9, copies=4, train=False) for dim, dv in ((32, 128), (64, 101), (128, 128))]
    + [case((F32,), [3000], 2, 1, dim, dv, sequences=9, copies=4, train=False) for dim, dv in ((32, 101), (64, 128))]
    + [case((BF16,), [6000], 2, kv, dim, dv, sequences=9, copies=2) for kv, dim, dv in ((2, 128, 60), (1, 101, 32))]
    + [case((BF16,), [6000], 2, kv, 128, 128, sequences=3, copies=4) for kv in (1, 2)]
    + [case((F32,), [3000], 2, 1, 128, 64, sequences=9, copies=2), case((F32,), [3000], 2, 2, 128, 30, sequences=9, copies=2)]
    # and packed.
    + [case((BF16,), [130, 0, 1, 700, 64, 500, 63, 1000] , 2, 1, 128, 101, sequences=16, copies=8, packed=True, train=False),
       case(ALL, [130, 1, 127, 128, 129, 700, 0, 63, 257, 256, 3, 900, 64], 2, 1, 128, 128, packed=True),
       case(SIXTEEN, [1, 700, 0, 63, 257, 900], 2, 2, 256, 100, packed=True),
       case((BF16,), [8000], 2, 1, 128, 128, copies=32, packed=True, train=False),
       case((BF16,), [8000], 2, 1, 128, 64, copies=16, packed=True), case((F32,), [4000], 2, 1, 64, 128, copies=32, packed=True, train=False)]
)


def passes(c, kind):
    """The lines that walk_plan.cpp reads, of the forward and of the backward pass's parts."""
    n = sum(c["lengths"])
    count = c["sequences"] * len(c["lengths"])
    tokens = c["sequences"] * n if c["packed"] else n
    heads, dim, dv = c["heads"] * c["copies"], c["dim"], c["value_dim"]
    line = lambda d, cols, together: (kind, c["packed"], count, tokens, heads, d, cols, together)  # noqa: E731
    found = [line(dim, dv, 1)]
    if c["train"]:
        found += [line(dv, dim, 3 if dim == dv else 2), line(dim, dv, 3 if dim == dv else 1)]
    return found
