"""Sizes that reach each launch form of the 4-bit products, for the host check that they do and the GPU tests
that compare them with float64: (x rows, weight rows, columns, geglu, (16-row tiles of x, accumulator registers,
row blocks of a workgroup, x in LDS)); the geglu form's two matrices take the place of two row blocks. Weight rows are no multiple of a workgroup's, so that its last row block
repeats; the fewest columns are one tile that is not full."""

FORMS = [
    (1, 8195, 160, False, (1, 1, 1, True)),
    (4, 100, 1152, True, (1, 1, 1, True)),
    (4, 40, 8224, False, (1, 2, 1, False)),  # x past what LDS keeps
    (5, 70, 160, False, (1, 2, 1, False)),
    (8, 100, 1152, True, (1, 2, 1, False)),
    (12, 1001, 96, False, (1, 4, 1, False)),
    (12, 8195, 160, False, (1, 4, 2, False)),
    (12, 16403, 32, False, (1, 4, 4, False)),
    (13, 16435, 1152, False, (1, 4, 4, False)),
    (9, 1001, 160, True, (1, 4, 1, False)),
    (16, 8211, 96, True, (1, 4, 2, False)),
    (40, 1001, 1152, False, (1, 4, 1, False)),
    (20, 4101, 160, False, (2, 4, 1, False)),
    (32, 8195, 96, False, (2, 4, 2, False)),
    (40, 2070, 1152, False, (2, 4, 1, False)),
    (17, 2070, 160, True, (2, 4, 1, False)),
    (32, 4133, 96, True, (2, 4, 1, False)),
    (64, 4101, 32, False, (4, 4, 1, False)),
    (65, 4101, 160, False, (4, 4, 2, False)),
    (64, 8195, 1152, False, (4, 4, 2, False)),
    (49, 2070, 96, True, (4, 4, 1, False)),
    (100, 4133, 160, True, (4, 4, 1, False)),
]
# Products of one matrix's rows that take different forms.
NEIGHBOURS = (8195, 1152, (1, 4, 5, 8, 12, 16, 20, 32, 40, 64, 65))
