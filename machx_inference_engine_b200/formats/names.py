"""Names in a GGUF file that are this engine's own: the scales beside a matrix of e4m3 codes (an I8 tensor), and the rows and the elements of K that share one."""
FP8_SCALES = ".fp8_scale"
FP8_BLOCK_ROWS, FP8_BLOCK_COLS = "machx.fp8.block_rows", "machx.fp8.block_cols"
