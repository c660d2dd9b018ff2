"""Which kernel of inner_prod_mxfp4 a call runs, by the rules of inner_prod_mxfp4_tc.cu and inner_prod_mxfp4_few.cu restated, and sizes that reach every one of them."""
SMEM, BLOCK, SM_COUNT = 227 * 1024, 128, 148          # bytes of a CTA's shared memory, bytes of K a stage, multiprocessors


def up(a, b):
    return -(-a // b)


def stages_of(bn, pair, split, residual):
    """The most stages that fit beside a kernel's staged outputs and the other CTAs' sums, and a stage's bytes."""
    warps = 16 if bn >= 128 else 8
    rows, scales = (bn // 2 if pair else bn), up(bn, 128)
    stage = 128 * BLOCK + rows * BLOCK + (1 + scales) * 1024
    fixed = 2048 + warps * (4096 if residual and split == 1 else 2048) + (split - 1) * 128 * 32 * 4
    return min(8, (SMEM - fixed) // stage)


def kernel_of(m, n, k, residual=False, floating=False):
    """("few", tokens of an MMA, CTAs a tile, whether it quantizes) or ("tiles", channels, CTAs that share a tile's K, whether a CTA has several tiles, whether it keeps weights)."""
    kblocks = up(up(k, 32) * 16, BLOCK)
    cluster = 1
    while cluster < 4 and 2 * cluster <= kblocks and up(n, 128) * cluster * 2 <= 2 * SM_COUNT:
        cluster *= 2
    if floating and m <= 16 and m * up(kblocks, cluster) <= 64 and up(kblocks, cluster) * (16 * BLOCK + 1024) <= 48 * 1024:
        return "few", 16, cluster, True
    if m <= 32 or (m <= 64 and up(k, 32) > 32):
        return "few", 16 if m <= 16 else 32 if m <= 32 else 64, cluster, False

    def clocks(bn, ctas):
        rounds = up(up(m, 128 * ctas) * up(n, bn), SM_COUNT // ctas)
        return rounds * (kblocks * 2 * (128 + bn // ctas) + 9 * bn + (ctas - 1) * 3500)

    def split_clocks(ctas):
        if up(m, 128) * up(n, 32 * ctas) * ctas > SM_COUNT or kblocks < ctas:
            return float("inf")
        return up(kblocks, ctas) * 2 * (128 + 32 * ctas) + 9 * 32 * ctas + 1000 * ctas

    c64, c128, pair, split2, split4 = clocks(64, 1), clocks(128, 1), clocks(256, 2), split_clocks(2), split_clocks(4)
    if min(split2, split4) < min(c64, c128, pair):
        return ("tiles", 128, 4, False, False) if split4 <= split2 else ("tiles", 64, 2, False, False)
    bn = 256 if pair < min(c64, c128) else 64 if c64 <= c128 else 128
    ctas = 2 if bn == 256 else 1
    tiles_m, tiles_n = up(m, 128 * ctas), up(n, bn)
    clusters = min(tiles_m * tiles_n, SM_COUNT // ctas)
    several = clusters < tiles_m * tiles_n
    if several and ctas == 1 and tiles_n <= 4:
        clusters -= clusters % tiles_n
    most = stages_of(bn, ctas == 2, 1, residual)
    stages = most if ctas == 2 else min(most, up(tiles_m * tiles_n, clusters) * kblocks)
    return "tiles", bn, 1, several, ctas == 1 and several and tiles_n <= 4 and kblocks <= stages


# (m, n, k), and what it reaches: without a residual, and with one where that is something else
FEW = [((1, 100, 200), ("few", 16, 1, False)), ((16, 4000, 500), ("few", 16, 2, False)), ((7, 1000, 4096), ("few", 16, 4, False)), ((2, 20000, 512), ("few", 16, 1, False)),
       ((20, 300, 256), ("few", 32, 1, False)), ((32, 300, 700), ("few", 32, 2, False)), ((25, 2000, 2048), ("few", 32, 4, False)), ((50, 20000, 1056), ("few", 64, 1, False)),
       ((64, 10000, 1100), ("few", 64, 2, False)), ((40, 1000, 4096), ("few", 64, 4, False))]
FLOATING = [((1, 100, 200), ("few", 16, 1, True)), ((16, 4000, 500), ("few", 16, 2, True)), ((5, 1000, 4096), ("few", 16, 4, True)), ((16, 300, 8192), ("few", 16, 4, False))]
WHOLE = [((40, 300, 300), ("tiles", 64, 1, False, False)), ((1000, 1000, 1000), ("tiles", 64, 1, False, False)), ((20000, 192, 4096), ("tiles", 64, 1, True, False)),
         ((9472, 256, 4096), ("tiles", 128, 1, False, False)), ((2048, 2048, 512), ("tiles", 128, 1, True, False)), ((600, 40000, 300), ("tiles", 128, 1, True, False))]
PAIRS = [((300, 9000, 8192), ("tiles", 256, 1, False, False)), ((2500, 2304, 4096), ("tiles", 256, 1, True, False))]
SPLIT = [((130, 512, 4112), ("tiles", 64, 2, False, False)), ((100, 4096, 4096), ("tiles", 64, 2, False, False)), ((90, 161, 8000), ("tiles", 64, 2, False, False)),
         ((128, 1024, 14336), ("tiles", 128, 4, False, False)), ((70, 300, 11008), ("tiles", 128, 4, False, False)), ((129, 130, 16384), ("tiles", 128, 4, False, False))]
KEPT = [((50000, 24, 500), ("tiles", 64, 1, True, True)), ((50000, 192, 256), ("tiles", 64, 1, True, True)), ((40001, 60, 700), ("tiles", 64, 1, True, True)),
        ((100352, 256, 64), ("tiles", 128, 1, True, True)), ((30000, 200, 1000), ("tiles", 128, 1, True, True)), ((33000, 384, 300), ("tiles", 128, 1, True, True)),
        ((40000, 100, 1200), ("tiles", 128, 1, True, True), ("tiles", 128, 1, True, False))]
ALL = FEW + WHOLE + PAIRS + SPLIT + KEPT
