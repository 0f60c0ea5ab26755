"""Sizes of the label fields' operators with the kernel that each takes (part of its name in the library): what the GPU tests
run, checked against what the library launches."""

# block products, m x n x k: tiles of 16 x (4 or so) rows a wave, by waves; odd sizes, a cut last block, more than four blocks
PRODUCTS = [
    (60, 301, 1100, "Li2ELi2ELi2ELi2E"),
    (1601, 1099, 1100, "Li4ELi4ELi2ELi2E"),
    (4001, 2050, 1100, "Li6ELi3ELi2ELi4E"),
    (2899, 2900, 1301, "Li6ELi3ELi2ELi4E"),
    (3900, 3901, 1100, "Li8ELi4ELi2ELi4E"),
    (3557, 2529, 1027, "Li8ELi4ELi2ELi4E"),
]

# linear layers, m x n x k
LINEARS = [
    (1, 32770, 300, "linear_few_kernelI{x}{out}Li2E"),
    (16, 32771, 300, "linear_few_kernelI{x}{out}Li2E"),
    (1, 50, 33000, "linear_few_kernelI{x}{out}Li1E"),   # two stretches of k
    (2, 50, 16500, "linear_few_kernelI{x}{out}Li1E"),
    (16, 333, 130, "linear_few_kernelI{x}{out}Li1E"),
    (500, 64, 257, "linear_head_kernelI{x}{out}Li4E"),
    (500, 128, 384, "linear_head_kernelI{x}{out}Li8E"),
    (500, 129, 128, "linear_head_kernelI{x}{out}Li12E"),
    (3001, 150, 257, "linear_head_kernelI{x}{out}Li12E"),  # the weight's three blocks do not fit at a time
    (500, 192, 384, "linear_head_kernelI{x}{out}Li12E"),
    (500, 193, 256, "linear_head_kernelI{x}{out}Li16E"),
    (40001, 150, 128, "linear_head_kernelI{x}{out}Li12E"),
    (300, 300, 300, "product_kernelI{out}Li4ELi4ELi2ELi2E"),
]

# distillation, rows x logits of float32, entries
DISTILLS = [
    (5, 1024, 1024, "distill_held_kernelIfLi64E"),     # entries that fill 64 KB of a workgroup's LDS, and the slots
    (9, 1025, 1023, "distill_held_kernelIfLi64E"),
    (200, 40000, 64, "distill_held_kernelIfLi1024E"),
    (200, 60001, 33, "distill_held_kernelIfLi1024E"),
    (300, 131072, 16, "distill_finish_kernelIf"),      # two batches of launches
]
