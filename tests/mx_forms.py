"""Shapes that reach each form of the kernels of microscaled products: what tests/test_mx_forms.py tells without a device and
tests/test_gpu_mx_forms.py runs."""
from __future__ import annotations

# Few rows, a kernel of their own: outputs for which a block takes 1, 2, 3, 4, 6 and 8 tiles of 16 (ending inside one), and
# more of them than 256 blocks take at a time.
TILES = [(1000, 1), (4090, 1), (4099, 2), (8200, 3), (12285, 3), (12300, 4), (16400, 6), (24500, 6), (24600, 8), (32760, 8), (40001, 8), (65530, 8)]
FEW = [1, 5, 16]

# ... whose fp32 rows' terms do not fit the LDS (M ceil(K / 128) above 321): several segments; the last two with more outputs than
# the blocks take at a time, so that every block cuts its rows again for the next ones.
SEGMENTS = [(11, 4096, 300), (16, 2600, 5000), (1, 49000, 600), (6, 8000, 1000), (16, 2570, 33000), (1, 42000, 33100)]

# both sides of the rules' borders: rows times inputs of 48 K, 64 K outputs, 16 rows
BORDERS = [((12, 4096, 200), (12, 4097, 200)), ((3, 16384, 130), (3, 16385, 130)), ((1, 49152, 70), (1, 49153, 70)),
           ((5, 96, 65536), (5, 96, 65537)), ((16, 300, 2000), (17, 300, 2000))]

# the other kernel: row blocks of 16, 32, 64 and 128 rows, of at most 256 blocks (double-buffered) and more, split and whole
BLOCKS = [(16, 4096, 300), (9, 60000, 100), (2, 256, 70000), (20, 4096, 500), (32, 700, 3000), (61, 768, 50257), (33, 11008, 4096),
          (300, 512, 27000), (300, 2050, 300), (1024, 300, 16400), (250, 130, 65600)]
