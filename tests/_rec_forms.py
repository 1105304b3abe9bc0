"""Shapes that take every form of the gated recurrence's kernels: how many steps a tile has, whether the
width is whole pieces of 8 bytes ("-") or not ("part"), and one tile, many, or a time axis cut into segments.
test_sequence.py holds the forms against the size queries, so that a changed rule cannot move a shape to
another form unseen; test_gpu_sequence.py runs them."""

STEPS = {"flat": 8, "short": 32, "wave": 64, "long": 256, "wide": 128, "slim": 64, "slim_long": 1024}

# (form, width, tiles, B, T, D) of fp32 rows, and of 16-bit rows
FORMS = {
    4: [
        ("flat", "-", "many", 8200, 20, 8), ("flat", "part", "many", 8200, 20, 7),
        ("short", "-", "one", 3, 20, 68), ("short", "part", "one", 3, 20, 67),
        ("wave", "-", "one", 2, 60, 132), ("wave", "part", "one", 2, 60, 131),
        ("wave", "-", "many", 170, 100, 264), ("wave", "part", "many", 170, 300, 131),
        ("long", "-", "one", 3, 200, 132), ("long", "part", "one", 3, 200, 131),
        ("long", "-", "many", 44, 1030, 68), ("long", "part", "many", 44, 1030, 67),
        ("long", "-", "cut", 2, 1300, 68), ("long", "part", "cut", 2, 1300, 67),
        ("wide", "-", "one", 2, 100, 1000), ("wide", "part", "one", 2, 100, 1001),
        ("wide", "-", "many", 160, 450, 40), ("wide", "part", "many", 160, 450, 39),
        ("wide", "-", "cut", 2, 700, 1000), ("wide", "part", "cut", 2, 700, 1001),
        ("slim", "-", "many", 300, 200, 12), ("slim", "part", "many", 300, 200, 13),
        ("slim_long", "-", "many", 140, 2100, 8), ("slim_long", "part", "many", 140, 2100, 7),
        ("slim_long", "-", "cut", 2, 5000, 8), ("slim_long", "part", "cut", 2, 5000, 7),
    ],
    2: [
        ("flat", "-", "many", 8200, 20, 8), ("flat", "part", "many", 8200, 20, 7),
        ("short", "-", "one", 3, 20, 68), ("short", "part", "one", 3, 20, 67),
        ("wave", "-", "one", 2, 60, 132), ("wave", "part", "one", 2, 60, 131),
        ("wave", "-", "many", 170, 100, 264), ("wave", "part", "many", 180, 300, 131),
        ("long", "-", "one", 3, 200, 132), ("long", "part", "one", 3, 200, 131),
        ("long", "-", "many", 130, 1030, 60), ("long", "part", "many", 130, 1030, 59),
        ("long", "-", "cut", 2, 1300, 132), ("long", "part", "cut", 2, 1300, 131),
        ("wide", "-", "one", 2, 100, 1000), ("wide", "part", "one", 2, 100, 1001),
        ("wide", "-", "many", 160, 450, 72), ("wide", "part", "many", 160, 450, 71),
        ("wide", "-", "cut", 2, 700, 1000), ("wide", "part", "cut", 2, 700, 1001),
        ("slim", "-", "many", 300, 200, 12), ("slim", "part", "many", 300, 200, 13),
        ("slim_long", "-", "many", 140, 2100, 8), ("slim_long", "part", "many", 140, 2100, 7),
        ("slim_long", "-", "cut", 2, 5000, 8), ("slim_long", "part", "cut", 2, 5000, 7),
    ],
}
