"""Batches that reach each variant of the paged attention's launches: the sizes, and
the launch that they are meant to get (checked on the CPU, run on the GPU)."""
from dataclasses import dataclass, field


@dataclass
class Variant:
    new: list
    lens: list
    heads: int
    kv_heads: int
    width: int       # entries of the page tables, 16 tokens each
    rows: int        # of a tile: 16 (k_attn_rows) or 128 (k_attn_chunk)
    parts: tuple     # fewest and most parts that a tile's keys are split into
    halves: bool     # whether two halves of a workgroup share a tile's keys
    dims: list = field(default_factory=lambda: [64, 80, 96, 128, 192, 256])
    window: int = 0

    def ids(self):
        return f"{self.rows}rows-{self.parts[0]}parts-{self.heads}heads-{'halves' if self.halves else 'one'}-w{self.window}"


# two halves a workgroup (up to 128 wide; 64 with three parts of q): 260 and 320 tiles and heads
HALVES = [Variant([150], [290], 130, 130, 40, 128, (1, 1), True, dims=[40, 64, 96, 128]),
          Variant([150, 0, 60, 1], [290, 9, 60, 200], 64, 64, 40, 128, (1, 1), True, dims=[64, 80, 128])]
# one workgroup a tile
WHOLE = [Variant([150], [290], 260, 260, 40, 128, (1, 1), False, dims=[64, 128]),
         Variant([150], [290], 130, 130, 40, 128, (1, 1), True, dims=[192, 256]),  # (no halves at this width)
         Variant([70, 200], [130, 300], 172, 86, 40, 128, (1, 1), False, dims=[64, 96, 200])]
# parts joined a row a thread, and a row a workgroup
PARTS = [Variant([40], [700], 4, 2, 64, 128, (2, 16), False), Variant([40, 45], [1900, 600], 2, 2, 130, 128, (2, 16), False),
         Variant([40], [5900], 2, 2, 375, 128, (17, 128), False), Variant([33, 70], [4500, 3000], 2, 1, 300, 128, (17, 128), False)]
# a window over several parts that hold keys
WINDOWS = [Variant([60], [3000], 2, 2, 190, 128, (4, 16), False, window=1000),
           Variant([300], [2500], 2, 2, 160, 128, (3, 16), False, window=700),
           Variant([150], [290], 130, 130, 40, 128, (1, 1), True, dims=[64, 128], window=40),
           Variant([150], [290], 260, 260, 40, 128, (1, 1), False, dims=[64, 128], window=40),
           Variant([150], [290], 130, 130, 40, 128, (1, 1), True, dims=[256], window=40)]
# few rows: one part, parts whose last workgroup joins them, in groups of threads or not
FEW = [Variant([1, 2], [90, 100], 4, 2, 7, 16, (1, 2), False), Variant([1], [3000], 4, 1, 188, 16, (2, 128), False),
       Variant([1, 1, 3], [900, 2000, 40], 16, 2, 130, 16, (2, 128), False),
       Variant([16], [3000], 2, 2, 200, 16, (2, 128), False, window=700)]
ALL = HALVES + WHOLE + PARTS + WINDOWS + FEW
