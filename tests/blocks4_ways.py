"""Sizes of products and linear layers in 4-bit blocks with the kernel that each takes (part of its name in the library)."""

# products, m x n x k: tiles of 16 x (4 or so) rows a wave, by waves; odd sizes, a cut last step, more than two steps
PRODUCTS = [
    (60, 301, 1100, "Li2ELi2ELi2ELi2E"),
    (33, 17, 31, "Li2ELi2ELi2ELi2E"),
    (300, 290, 255, "Li2ELi2ELi2ELi2E"),
    (300, 290, 4100, "Li2ELi2ELi2ELi2E"),
    (1601, 1099, 1100, "Li2ELi2ELi2ELi2E"),
    (1901, 2300, 1301, "Li4ELi4ELi2ELi2E"),
    (20000, 257, 128, "Li4ELi4ELi2ELi2E"),
    (4001, 2050, 1100, "Li6ELi4ELi2ELi3E"),
    (2899, 2900, 1301, "Li6ELi4ELi2ELi3E"),
    (3900, 3901, 1100, "Li8ELi4ELi2ELi4E"),
    (3557, 2529, 1027, "Li8ELi4ELi2ELi4E"),
]

# linear layers, m x n x k, the rows' bytes an element and the kernel
LINEARS = [
    (1, 32771, 300, 2, "linear4_few_kernelI{x}{out}"),
    (16, 4099, 300, 4, "linear4_few_kernelI{x}{out}"),
    (2, 50, 16384, 4, "linear4_few_kernelI{x}{out}"),
    (2, 50, 16385, 4, "product4_kernelI{out}Li2ELi2ELi2ELi2E"),
    (16, 333, 130, 2, "linear4_few_kernelI{x}{out}"),
    (1, 4100, 32768, 2, "linear4_few_kernelI{x}{out}"),
    (2, 4100, 16385, 2, "product4_kernelI{out}Li2ELi2ELi2ELi2E"),
    (17, 40, 96, 2, "product4_kernelI{out}Li2ELi2ELi2ELi2E"),
    (4096, 64, 128, 2, "linear4_head_kernelI{x}{out}Li4E"),
    (4100, 7, 33, 4, "linear4_head_kernelI{x}{out}Li4E"),
    (8201, 65, 257 - 1, 2, "linear4_head_kernelI{x}{out}Li10E"),
    (20001, 150, 128, 2, "linear4_head_kernelI{x}{out}Li10E"),
    (5003, 160, 64, 4, "linear4_head_kernelI{x}{out}Li10E"),
    (5003, 128, 64, 2, "linear4_head_kernelI{x}{out}Li10E"),
    (12301, 193, 300, 2, "linear4_head_kernelI{x}{out}Li16E"),
    (4999, 256, 128, 4, "linear4_head_kernelI{x}{out}Li16E"),
    (16390, 16, 500, 2, "linear4_head_kernelI{x}{out}Li4E"),
    (5000, 257, 128, 2, "product4_kernelI{out}Li2ELi2ELi2ELi2E"),
    (300, 300, 300, 2, "product4_kernelI{out}Li2ELi2ELi2ELi2E"),
    (2333, 3001, 1100, 2, "product4_kernelI{out}Li4ELi4ELi2ELi2E"),
]
