"""Grouped products whose sizes lead to each of the tile kernels: (kind, bytes that every row starts on, rows, groups, channels, values, form).

The forms are pb_linear_form's: 3 tiles of 64 x 64, 4 of 128 x 128, 5 of 128 x 128 with waves of 64 x 64, 6 of 256 x 256.  Every one that a grouped
product of that type and alignment takes, once over a few groups and once over more than the 64 that a wave looks at together.  (Tiles of 128
x 128 with eight waves, 4, are chosen for grouped products in 8 and 16 bits only, and with rows on 4 bytes for dense ones alone; 256 x 256 needs rows
on 16 bytes and no f32.)"""

SIZE = {"f32": 4, "bf16": 2, "f16": 2, "i8": 1}
TYPE = {"f32": 0, "bf16": 1, "f16": 2, "i8": 3}
ALIGN = {"f32": (16, 4), "bf16": (16, 4, 2), "f16": (16, 4, 2), "i8": (16, 4, 1)}

_F32 = [(16, 243, 7, 1868, 121, 3), (16, 219, 66, 526, 129, 3), (16, 4993, 5, 2387, 125, 5), (16, 5031, 66, 2548, 125, 5),
        (4, 283, 7, 1630, 121, 3), (4, 216, 66, 518, 127, 3), (4, 4742, 3, 2432, 121, 5), (4, 6417, 97, 2029, 127, 5)]
_BITS16 = [(16, 8225, 5, 37, 179, 3), (16, 349, 97, 175, 185, 3), (16, 8278, 5, 478, 229, 4), (16, 8830, 130, 240, 473, 4), (16, 1926, 3, 2558, 171, 5),
           (16, 8955, 130, 379, 205, 5), (16, 8878, 3, 2968, 215, 6), (16, 8863, 66, 442, 1235, 6), (4, 201, 7, 2168, 171, 3), (4, 205, 66, 548, 173, 3),
           (4, 6614, 7, 639, 171, 5), (4, 8303, 97, 356, 191, 5), (2, 8917, 3, 36, 219, 3), (2, 302, 97, 241, 191, 3), (2, 7456, 3, 478, 203, 4),
           (2, 8765, 130, 207, 363, 4), (2, 1615, 3, 2815, 173, 5), (2, 8958, 130, 346, 171, 5)]
_I8 = [(16, 8542, 3, 36, 273, 3), (16, 340, 97, 175, 323, 3), (16, 8513, 7, 353, 731, 4), (16, 8714, 130, 222, 905, 4), (16, 2539, 11, 2006, 277, 5),
       (16, 8288, 97, 494, 283, 5), (16, 7899, 3, 2973, 521, 6), (16, 8600, 66, 950, 1337, 6), (4, 385, 11, 1210, 279, 3), (4, 523, 130, 240, 293, 3),
       (4, 4120, 3, 1096, 279, 5), (4, 8802, 130, 348, 297, 5), (1, 229, 7, 1765, 271, 3), (1, 425, 130, 175, 313, 3), (1, 8283, 3, 358, 537, 4),
       (1, 8950, 130, 233, 703, 4), (1, 4693, 11, 1027, 277, 5), (1, 8967, 130, 355, 277, 5)]
CASES = [(kind, *c) for kind, cases in (("f32", _F32), ("bf16", _BITS16), ("f16", _BITS16), ("i8", _I8)) for c in cases]


def row_stride(kind: str, k: int, align: int) -> int:
    """the least stride of at least k elements whose rows start on `align` bytes and on no larger power of two up to 16"""
    size, ld = SIZE[kind], k
    while (ld * size) % align or (align < 16 and (ld * size) % (2 * align) == 0):
        ld += 1
    return ld
