"""Sizes (M, K, N) that reach every form of the 4-bit product and its gradient (csrc/mx4.hip), with the form that each is to take: kind, rows and
columns of a tile, waves along K / scales of four stages at once / rows of odd length, and whether the sum is split over blocks.  The CPU
test holds the choice to this list, so that new step costs cannot take a form out of the GPU test's sight unnoticed."""
TILES, DIRECT, TILES4, GRAD = 0, 1, 2, 3
PRODUCT = [
    ('f32', (1, 27, 5), (TILES, 16, 64, 0, False)), ('f32', (3, 6098, 33), (TILES, 16, 64, 0, True)),
    ('f32', (2050, 100, 328), (TILES, 32, 128, 0, False)), ('f32', (244, 4000, 130), (TILES, 32, 128, 0, True)),
    ('f32', (130, 100, 20001), (TILES, 64, 128, 0, False)), ('f32', (257, 12000, 260), (TILES, 64, 128, 0, True)),
    ('f32', (209, 100, 32559), (TILES, 64, 256, 0, False)), ('f32', (1000, 4000, 2001), (TILES, 64, 256, 0, True)),
    ('f32', (1, 4096, 4096), (DIRECT, 16, 16, 8, False)), ('f32', (12, 2000, 2049), (DIRECT, 16, 16, 8, False)),
    ('f32', (16, 1100, 1500), (DIRECT, 16, 16, 8, False)), ('f32', (8, 1024, 1023), (DIRECT, 16, 16, 8, False)),
    ('f32', (16, 800, 65), (DIRECT, 16, 32, 4, False)), ('f32', (1, 2448, 8192), (DIRECT, 16, 32, 8, False)),
    ('bf16', (1, 27, 5), (TILES, 16, 64, 0, False)), ('bf16', (3, 6098, 33), (TILES, 16, 64, 0, True)),
    ('bf16', (17, 100, 16401), (TILES, 32, 128, 0, False)), ('bf16', (200, 4000, 130), (TILES, 32, 128, 0, True)),
    ('bf16', (1000, 27, 1100), (TILES, 64, 128, 0, False)), ('bf16', (300, 8192, 130), (TILES, 64, 128, 0, True)),
    ('bf16', (207, 100, 32717), (TILES, 64, 256, 0, False)), ('bf16', (1000, 33000, 2001), (TILES, 64, 256, 0, True)),
    ('bf16', (1, 4096, 4096), (DIRECT, 16, 16, 8, False)), ('bf16', (12, 2000, 2049), (DIRECT, 16, 16, 8, False)),
    ('bf16', (16, 1500, 1001), (DIRECT, 16, 16, 8, False)), ('bf16', (3, 3000, 513), (DIRECT, 16, 16, 8, False)),
    ('mx4', (1, 1024, 7), (DIRECT, 16, 16, 8, False)), ('mx4', (5, 20000, 7), (DIRECT, 16, 16, 8, True)),
    ('mx4', (3, 520, 70), (DIRECT, 16, 32, 4, False)), ('mx4', (16, 1024, 8192), (DIRECT, 16, 32, 8, False)),
    ('mx4', (9, 130, 33), (DIRECT, 16, 64, 2, False)), ('mx4', (16, 520, 16384), (DIRECT, 16, 64, 4, False)),
    ('mx4', (2, 27, 5), (DIRECT, 16, 128, 1, False)), ('mx4', (11, 130, 32768), (DIRECT, 16, 128, 2, False)),
    ('mx4', (18, 1024, 33), (DIRECT, 32, 16, 8, False)), ('mx4', (31, 20000, 7), (DIRECT, 32, 16, 8, True)),
    ('mx4', (17, 520, 70), (DIRECT, 32, 32, 4, False)), ('mx4', (30, 1024, 8192), (DIRECT, 32, 32, 8, False)),
    ('mx4', (20, 130, 33), (DIRECT, 32, 64, 2, False)), ('mx4', (18, 520, 16385), (DIRECT, 32, 64, 4, False)),
    ('mx4', (32, 27, 129), (DIRECT, 32, 128, 1, False)), ('mx4', (18, 130, 32769), (DIRECT, 32, 128, 2, False)),
    ('mx4', (48, 1024, 33), (DIRECT, 64, 16, 8, False)), ('mx4', (33, 20000, 7), (DIRECT, 64, 16, 8, True)),
    ('mx4', (50, 520, 70), (DIRECT, 64, 32, 4, False)), ('mx4', (48, 1024, 8193), (DIRECT, 64, 32, 8, False)),
    ('mx4', (64, 130, 33), (DIRECT, 64, 64, 2, False)), ('mx4', (48, 520, 16385), (DIRECT, 64, 64, 4, False)),
    ('mx4', (33, 27, 129), (DIRECT, 64, 128, 1, False)), ('mx4', (48, 130, 32769), (DIRECT, 64, 128, 2, False)),
    ('mx4', (129, 384, 264), (TILES4, 128, 128, 0, False)), ('mx4', (65, 12000, 70), (TILES4, 128, 128, 0, True)),
    ('mx4', (100, 1024, 200), (TILES4, 128, 128, 1, False)), ('mx4', (244, 6098, 328), (TILES4, 128, 128, 1, True)),
    ('mx4', (300, 100, 33000), (TILES4, 256, 256, 0, False)), ('mx4', (1000, 20000, 16400), (TILES4, 256, 256, 0, True)),
    ('mx4', (2050, 1000, 6001), (TILES4, 256, 256, 1, False)),
]
GRADIENT = [
    ('f32', (3, 27, 5), (GRAD, 16, 128, 0, False)), ('f32', (1, 33, 1100), (GRAD, 16, 128, 0, True)),
    ('f32', (5, 33000, 7), (GRAD, 16, 256, 0, False)), ('f32', (257, 130, 2000), (GRAD, 16, 256, 0, True)),
    ('f32', (17, 33000, 33), (GRAD, 32, 256, 0, False)), ('f32', (300, 300, 4096), (GRAD, 32, 256, 0, True)),
    ('bf16', (3, 27, 6), (GRAD, 16, 128, 0, False)), ('bf16', (3, 128, 32768), (GRAD, 16, 128, 0, True)),
    ('bf16', (5, 33000, 8), (GRAD, 16, 256, 0, False)), ('bf16', (257, 130, 2000), (GRAD, 16, 256, 0, True)),
    ('bf16', (2050, 300, 64), (GRAD, 64, 128, 0, False)), ('bf16', (257, 33, 6000), (GRAD, 64, 128, 0, True)),
    ('bf16', (2050, 1500, 7), (GRAD, 64, 128, 1, False)), ('bf16', (1000, 33, 3101), (GRAD, 64, 128, 1, True)),
]
