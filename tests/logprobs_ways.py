"""Rows x logits, alternatives and the kernel that each takes (part of its name in the library), by the logits' type."""


def _ways(t, wide):
    k = 1 if wide else 2  # elements of 4 bytes
    return [
        (5, 3, 2, f"held_kernelI{t}Li8ELi1E"),
        (33, 41, 3, f"held_kernelI{t}Li8ELi2E"),
        (300, 75, 8, f"held_kernelI{t}Li8ELi3E"),
        (33, 80, 3, f"held_kernelI{t}Li8ELi3E"),
        (9, 120, 8, f"held_kernelI{t}Li8ELi4E"),
        (301, 150, 3, f"held_kernelI{t}Li8ELi5E"),
        (40, 191, 6, f"held_kernelI{t}Li8ELi6E"),
        *([(9, 256, 8, f"held_kernelI{t}Li8ELi8E"), (30, 201, 8, f"held_kernelI{t}Li8ELi8E"),
           (37, 361, 5, f"held_kernelI{t}Li16ELi3E")] if not wide else [(37, 201, 5, f"held_kernelI{t}Li16ELi4E")]),
        (21, 250 * k + 1, 5, f"held_kernelI{t}Li16ELi4E"),
        (6, 150, 9, f"held_kernelI{t}Li8ELi5E"),
        (70, 150, 64, f"held_kernelI{t}Li8ELi5E"),
        (11, 14, 14, f"held_kernelI{t}Li8ELi1E"),
        (37, 251 * k, 16 // (3 - k), f"held_kernelI{t}Li16ELi4E"),
        (37, 300 * k, 3, f"held_kernelI{t}Li16ELi5E"),
        (19, 383 * k, 8, f"held_kernelI{t}Li16ELi6E"),
        *([(19, 1024, 8, f"held_kernelI{t}Li16ELi8E"), (40, 801, 5, f"held_kernelI{t}Li16ELi8E")] if not wide else []),
        (6, 255 * k, 17, f"held_kernelI{t}Li64ELi1E"),
        (70, 250 * k, 40, f"held_kernelI{t}Li64ELi1E"),
        (5, 1021 * k, 64, f"held_kernelI{t}Li64ELi4E"),
        (66, 700 * k, 5, f"held_kernelI{t}Li64ELi4E"),
        (4, 1500 * k + 1, 64, f"held_kernelI{t}Li256ELi4E"),
        (3, 4111 * k, 20, f"slices_kernelI{t}Li4E"),
        (193, 6001 * k, 33, f"held_kernelI{t}Li256ELi8E"),
        (192, 16001 * k, 8, f"held_kernelI{t}Li256ELi16E"),
        (193, 30011 * k, 20, f"held_kernelI{t}Li512ELi16E"),
        (192, 65000 * k, 64, f"held_kernelI{t}Li1024ELi16E"),
        (1, 65537 * k, 20, f"slices_kernelI{t}Li4E"),
        (200, 90001 * k, 7, f"slices_kernelI{t}Li16E"),
    ]


WAYS = {"f": _ways("f", True), "DF16b": _ways("DF16b", False), "DF16_": _ways("DF16_", False)}
