"""Sizes of the 8-bit linear and the kernel that takes each on 148 SMs, all free: (m, n, k) to (kernel, tokens of a tile, what else):

("rows", tokens, weight rows a warp), ("few", tokens of a tile, CTAs that share K), ("pairs", tokens of a tile, how the last round runs)."""
SIZES = {
    (1, 6145, 4096): ("rows", 1, 2), (1, 4737, 16): ("rows", 1, 2), (1, 1030, 4112): ("rows", 1, 1),
    (2, 2001, 528): ("rows", 2, 1), (2, 4099, 1040): ("rows", 2, 2),
    (3, 65, 16): ("rows", 4, 2), (4, 4097, 2064): ("rows", 4, 2), (3, 4801, 1040): ("rows", 4, 4), (4, 4803, 2064): ("rows", 4, 4),
    (5, 65, 16): ("few", 16, 1), (5, 4705, 1168): ("few", 16, 2), (5, 67, 880): ("few", 16, 4), (5, 67, 944): ("few", 16, 8),
    (18, 9473, 16): ("few", 32, 1), (17, 5183, 1744): ("few", 32, 2), (17, 2201, 960): ("few", 32, 4), (18, 995, 912): ("few", 32, 8),
    (33, 9603, 16): ("few", 64, 1), (35, 5155, 3232): ("few", 64, 2), (35, 2867, 1824): ("few", 64, 4), (33, 1671, 1456): ("few", 64, 8),
    (65, 9523, 16): ("few", 128, 1), (68, 6307, 4928): ("few", 128, 2), (68, 3129, 2880): ("few", 128, 4), (70, 1867, 2800): ("few", 128, 8),
    (258, 15706, 16): ("pairs", 128, "whole"), (259, 15707, 272): ("pairs", 128, "whole"),
    (390, 11055, 16): ("pairs", 128, "halves"), (1000, 5000, 528): ("pairs", 128, "halves"),
    (194, 9797, 16): ("pairs", 256, "whole"), (600, 5003, 2064): ("pairs", 256, "whole"),
    # more tiles than pairs: whole ones first, then the rest as halves, the last of them with a single token
    (129, 19534, 16): ("pairs", 256, "halves"), (900, 5501, 1040): ("pairs", 256, "halves"), (2600, 2300, 1296): ("pairs", 256, "halves"),
}
