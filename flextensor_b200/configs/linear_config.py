"""Shapes of the feed-forward operators of language models (no counterpart in the reference).

``linear_shapes``: (tokens, N, K, activation, gated) from one token to a long batch.
``expert_shapes``: (tokens, experts, top_k, hidden, inner) of an expert feed-forward block.
"""
linear_shapes = [
    (1, 4096, 4096, "none", False),
    (64, 4096, 4096, "gelu", False),
    (2048, 2048, 2048, "silu", True),
    (4096, 4096, 4096, "none", False),
]

expert_shapes = [
    (8, 64, 8, 2048, 1024),
    (4096, 32, 4, 2048, 2048),
]
