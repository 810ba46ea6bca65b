"""FlashAct for MI355X: the flow-matching denoise loop of VLA action experts on gfx950.

Modules:
  pi05       -- pi0.5 (Gemma-300M-shaped) expert: ``launch`` (drop-in for src/pi05 ``mk_v6.launch``),
                packing, RoPE table, KV compaction, modulation precompute.
  prefill    -- the backbone: prefix prefill, packed prompts, further tokens on 8-bit caches and 4-bit weights.
  attention  -- attention in which every query has its own span of keys.
  kv8        -- the 8-bit K/V cache: rows in and out, and attention of the newest tokens over it.
  w4         -- products of a few rows with 4-bit weights.
  synthetic  -- seeded synthetic weights and inputs of the benchmark shapes.
  build      -- builds libflashact_mi355x.so in-tree with hipcc (gfx950).
"""
__all__ = ["pi05", "prefill", "attention", "kv8", "w4", "synthetic", "build"]
