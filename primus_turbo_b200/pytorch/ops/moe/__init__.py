from .few_tokens import moe_few_tokens  # noqa: F401
from .permutation import token_permute, token_unpermute  # noqa: F401
from .router import topk_router, topk_routing_map  # noqa: F401

__all__ = ["token_permute", "token_unpermute", "topk_router", "topk_routing_map", "moe_few_tokens"]
