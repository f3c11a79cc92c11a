"""Shapes of the MXFP4 and 8-bit cache tests that are there for the kernel they take: test_lowbit_host.py holds them against
what the library says it launches, the GPU tests run them."""

# M, N, K of quantised rows. Few rows: one, two and four tiles of 16, four and eight waves
ROWS = [(9, 100, 1000), (16, 64, 4304), (20, 60, 768), (32, 130, 2304), (40, 90, 520), (200, 516, 2304), (600, 768, 256)]
# tiles through the LDS ring: rows and columns that end inside a tile, N a multiple of 8 (16-byte stores) and odd, every
# remainder of the four steps that share a scale register; of 128-row tiles more than workgroups
TILES = [(500, 2040, 1152), (512, 2045, 650), (1280, 768, 768), (512, 2048, 2048),  # 64 x 64
         (730, 2304, 768), (729, 2299, 1152), (700, 2304, 2048),                    # 64 x 128
         (4000, 4304, 1152), (3900, 4301, 641), (794, 8192, 2048),                  # 128 x 128
         (2600, 3336, 384), (700, 1001, 300), (2600, 3333, 512),                    # 128 x 128, two steps in the ring
         (4096, 8184, 640), (4100, 8190, 1152), (4033, 8192, 770)]                  # 128 x 256
# M, N, K of bf16 rows quantised inside the launch: one, up to four, up to eight rows, K a multiple of 8 or not, four and eight
# waves
FEW = [(1, 130, 1152), (1, 100, 4304), (3, 60, 768), (4, 64, 2304), (7, 72, 2048), (8, 50, 2056), (6, 40, 1001), (5, 33, 2100)]

# sequences' lengths, key heads, group, head dim, queries, causal_from, capacity (0: the longest). One for each kernel with and
# without a join; runs of more than 64 blocks, whose scales come in a second load
ATTENTION = [
    ((700, 0, 1, 64, 699) * 4, 16, 1, 64, 1, None, 0), ((4000, 5, 4000, 1111) * 5, 16, 1, 64, 1, None, 0),       # 16 rows, 4 waves
    ((700, 0, 1, 64, 699) * 4, 16, 2, 128, 1, None, 0), ((4000, 5, 4000, 1111) * 5, 16, 1, 128, 2, 0, 0),
    ((130, 77), 3, 4, 64, 1, None, 200), ((5000, 3), 2, 2, 64, 7, 0, 0),                                         # 16 rows, 8 waves
    ((130, 77), 3, 4, 128, 1, None, 200), ((5000, 3), 2, 2, 128, 7, 0, 0),
    ((150,), 2, 1, 64, 100, 0, 300), ((6000,), 4, 1, 64, 70, 0, 0), ((5000,), 70, 1, 64, 64, 50, 0),             # 32 rows
    ((150,), 2, 1, 128, 100, 0, 300), ((6000,), 4, 4, 128, 30, 0, 0), ((5000,), 70, 1, 128, 64, 50, 0),
    ((5000,), 48, 1, 64, 256, 0, 0), ((16500,), 2, 1, 64, 60, None, 0),                                          # 64 rows
    ((5000,), 48, 1, 128, 256, 0, 0), ((16500,), 2, 3, 128, 20, 0, 0),
    ((4500,), 192, 1, 64, 70, 0, 0), ((16500,), 2, 2, 64, 60, 0, 0),                                             # 128 rows, 2 key waves
    ((4500,), 192, 1, 128, 70, 0, 0), ((16500,), 2, 8, 128, 20, 0, 0),
    ((4500,), 512, 1, 64, 100, 0, 0), ((4500, 130, 4444, 1), 8, 4, 128, 512, 0, 0),                              # 128 rows
]

# key heads, group, head dim, queries: each kernel over one sequence of 150 keys in a cache of 200
MASKED = [(2, 1, 64, 20), (200, 1, 64, 20), (2, 1, 128, 20), (200, 1, 128, 20), (2, 1, 64, 70), (2, 1, 128, 70), (100, 1, 64, 70),
          (100, 1, 128, 70), (192, 1, 64, 70), (100, 2, 128, 70), (512, 1, 64, 70), (256, 2, 128, 70)]
