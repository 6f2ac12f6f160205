"""Products by the kernel they are meant to reach, for the tests on the host (which kernel it is) and on the GPU (what it
computes)."""

# K past two spans of scales (a span: 1024 elements): whole steps of 256, a half step at the end, rows of scales that are no
# multiple of 16 bytes, an odd K, many spans
LONG_K = [2304, 2432, 2560, 2601, 2690, 8200]
TILES = {"amos_mx_gemm_tile<32x64>": [(300, 520), (40, 4500)], "amos_mx_gemm_tile<64x64>": [(520, 1100), (1000, 700)],
         "amos_mx_gemm_tile<128x128>": [(1500, 1700), (2100, 1000)], "amos_mx_gemm_tile<128x256>": [(2304, 2304), (2310, 2250)],
         "amos_mx_gemm_tile<256x256>": [(3000, 2900), (3100, 3005)]}
LONG = [(kernel, M, N, K) for kernel in TILES for i, K in enumerate(LONG_K) for M, N in [TILES[kernel][i % 2]]]
# up to 16 tokens on one, two and three blocks of 16 rows of B a workgroup: whole and ragged blocks, a turn and more of K a wave
FEW = [(rt, M, N, K) for rt, M, N, K in [(1, 3, 4090, 700), (2, 1, 5000, 600), (2, 16, 8190, 1100), (2, 7, 4112, 9001), (2, 5, 8192, 128),
                                         (3, 9, 12200, 4100), (3, 16, 12288, 520), (3, 1, 8200, 33), (3, 12, 8300, 9100)]]
# of those, what takes dense rows without a launch in front: K up to 4096, 32 KB of rows
FUSED = {"float32": lambda M, K: M * K * 4 <= 32768 and K <= 4096, "float16": lambda M, K: M * K * 2 <= 32768 and K <= 4096,
         "bfloat16": lambda M, K: M * K * 2 <= 32768 and K <= 4096}
