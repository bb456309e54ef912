"""Attentions over the paged K/V cache, one or more to each kernel that a call may choose: test_pages_forms.py looks at what
is launched, test_gpu_pages_forms.py at what comes out."""
import moert

TYPES = {moert.F32: 0, moert.F16: 1, moert.BF16: 2}  # of rows, as the kernels number them

# name: call; sequences, KV heads, page, pages, pages of a sequence; query heads; rows before; new rows; kernels
FORMS = {
    "positions, many splits": ("attend", (3, 2, 64, 80, 200), 6, [2999, 39, 1099], [1, 1, 1], ["cols", "join 16"]),
    "positions, eight splits": ("attend", (8, 4, 32, 200, 128), 8, [1200, 0, 31, 500, 128, 129, 1000, 700], [1] * 8,
                                ["cols", "join_few 16"]),
    "positions, streamed": ("attend", (2, 8, 256, 200, 100), 16, [699, 33], [1, 1], ["cols streamed", "join 16"]),
    "few rows, many splits": ("prompt", (1, 1, 64, 50, 100), 4, [2900], [8], ["cols", "join 16"]),
    "few rows, two splits": ("prompt", (4, 8, 64, 60, 100), 16, [900, 100, 0, 700], [15, 1, 20, 24], ["cols", "join_few 16"]),
    "many rows, many splits": ("prompt", (1, 1, 64, 80, 200), 4, [4000], [50], ["tiles", "join 128"]),
    "many rows, six splits": ("prompt", (4, 8, 64, 60, 100), 16, [800, 0, 300, 1000], [100, 130, 1, 169],
                              ["tiles", "join_few 128"]),
    "many rows": ("prompt", (2, 2, 64, 40, 15), 6, [333, 0], [200, 150], ["tiles"]),
}


def kernel(what, d, dtype):
    """What the name of a kernel has in it."""
    name, *arg = what.split()
    args = [d, TYPES[dtype]] + ([int(arg[0])] if arg and arg[0].isdigit() else [])
    flag = "" if name != "cols" else "Lb1E" if arg == ["streamed"] else "Lb0E"
    return "k_pages_" + name + "I" + "".join(f"Li{x}E" for x in args) + flag + "E"
