"""nerf_amd: the NeRF render path of dgsmith7/nerf-dbr on MI355X (gfx950) HIP kernels.

weights      -- NeRFModel state-dict schema, checkpoints, the synthetic checkpoint
runtime      -- ctypes binding of libnerf_mi355x.so (include/nerf_mi355x.h)
operators    -- rotary positions with several axes, the gated feed-forward block and its gradients
optim        -- AdamW over many tensors, moments in 32 or 8 bits
distributed  -- row-band sharding + RCCL all-gather across one node's GPUs
benchmark    -- plugin interface, MI355XRenderer, benchmark suite
"""
__version__ = "0.1.0"
