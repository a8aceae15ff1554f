"""Library kernels (used by ``tilelang.models``).

* ``gemm.linear``        -- y = x W^T (MFMA GEMM, tiles picked by problem size)
* ``norm.rms_norm``      -- fused RMSNorm * weight (row in registers)
* ``norm.add_rms_norm_quant`` -- residual addition + RMSNorm + e4m3 output with scales, one pass
* ``quant.act_quant``    -- per-128-group fp8 (e4m3) activation quantisation with fp32 scales
* ``dsa``                -- DeepSeek sparse attention: sparse MLA, lightning indexer, top-k selector
* ``moe``                -- grouped-GEMM SwiGLU experts and token packing
* ``kv_cache``           -- e4m3 paged key/value cache (a scale per page and head): append, attention
* ``beam``               -- beam search: selection over beams and vocabulary, reordering of states

``add_rms_norm_quant``, ``kv_cache`` and ``beam`` are hand-written HIP kernels (``csrc/ops``, compiled ahead of
time into ``tilelang._tl_ops``); the others are programs of the tile DSL.
"""
