"""Matrices whose rows the forward pass gives several packs of 16 bytes a lane: more rows than the chip holds at a pack a lane.  Which kernel
a size takes is looked up in the launches themselves (test_rows_host.py), so a rule that changes cannot take one out of the tests' reach."""
import torch

CODES = {torch.float32: 0, torch.float64: 1, torch.float16: 2, torch.bfloat16: 3}  # cgnn_dtype
LANES = 1 << 19  # that the chip holds at once; 16-bit rows of more than 256 packs: four times as many

# (lanes, packs a lane): packs of the narrowest and of a wide row
SPREAD = {(1, 2): (2, 2), (1, 3): (3, 3), (2, 2): (4, 4), (2, 3): (5, 6), (4, 2): (7, 8), (4, 3): (9, 12), (8, 2): (13, 16), (8, 3): (17, 24),
          (16, 2): (25, 32), (16, 3): (33, 48), (32, 2): (49, 64), (32, 3): (65, 96), (64, 2): (97, 128), (64, 3): (129, 192),
          (64, 4): (193, 256), (64, 5): (257, 320), (128, 3): (321, 383), (256, 2): (385, 512)}


def many(dtype):
    """[(lanes, packs), rows, width]: for each a wide row of whole packs and the narrowest, one element in its last pack."""
    elements = 16 // torch.empty((), dtype=dtype).element_size()
    shapes = []
    for shape, (fewest, most) in SPREAD.items():
        for packs, width in ((most, most * elements), (fewest, (fewest - 1) * elements + 1)):
            lanes = 1 << (packs - 1).bit_length()
            rows = LANES * (4 if elements == 8 and packs > 256 else 1) // lanes + 3
            shapes.append((shape, rows, width))
    return shapes
