"""Sizes (tokens, channels, K) of the fp4 product by the kernels they run on a GPU of 148 SMs: a CPU test holds the lists to the
library's choice, so that a change of the choice cannot leave a path without its test unnoticed."""
SMS = 148

# the CTA-pair kernel, at least three rounds of tiles and more steps of K than its ring has stages: accumulators that overlap, the
# ring wrapping inside a tile and from one tile to the next. Rows of the result on 32 bytes, on 16, and on neither.
PAIR_ROUNDS = [(1100, 13008, 3104), (700, 19000, 1824), (1037, 12007, 2080), (2049, 7003, 4128)]
# whole rounds by the pair kernel, the columns that are left by the few-token kernel behind it
TWO_LAUNCHES = [(512, 9504, 8224), (257, 19001, 8224), (1000, 4994, 8224), (700, 12776, 8480)]
# the few-token kernel for more than one block of 128 tokens
FEW_TOKEN_BLOCKS = [(300, 9600, 1056), (150, 2050, 11008)]
# one round of the pair kernel: tiles of 128 channels, of 256
PAIR_ONE_ROUND = [(256, 1024, 2048), (1024, 4100, 1056)]
