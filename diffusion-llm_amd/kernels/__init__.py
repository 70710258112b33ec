"""MI355X (gfx950) BD3-LM attention kernels behind the reference's
`kernels/` module interface:

    kernels.BlockSparseFlashAttention.BlockSparseFlashAttention.apply(q, k, v, block_size)
    kernels.BlockSparseDecodeAttention.block_sparse_decode_attention(q, k, v, block_size)
    kernels.SplitKVDecodeAttention.split_kv_decode_attention(q, k, v, block_size)

and, for sequences of different lengths, kernels.paged (a paged KV cache, its
attention) with kernels.sampling.adjust_logits.

Each call lands in libbd3attn.so (hand-written HIP for gfx950) through the
C ABI of include/bd3attn.h.
"""
