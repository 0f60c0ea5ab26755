"""Sizes of products and linear layers in 4-bit blocks with the kernel that each takes (part of its name in the library)."""

# products, m x n x k: tiles of 16 x (4 or so) rows a wave, by waves; odd sizes, a cut last step, more than two steps
PRODUCTS = [
    (60, 301, 1100, "Li2ELi2ELi2ELi2E"),
    (33, 17, 31, "Li2ELi2ELi2ELi2E"),
    (1601, 1099, 1100, "Li4ELi4ELi2ELi2E"),
    (300, 290, 255, "Li4ELi4ELi2ELi2E"),
    (4001, 2050, 1100, "Li6ELi4ELi2ELi3E"),
    (2899, 2900, 1301, "Li6ELi4ELi2ELi3E"),
    (3900, 3901, 1100, "Li8ELi4ELi2ELi4E"),
    (3557, 2529, 1027, "Li8ELi4ELi2ELi4E"),
]
