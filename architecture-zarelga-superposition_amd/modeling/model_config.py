"""MoE fields of the reference's ModelConfig (modeling/model_config.py:45-185).

Only the fields the MoE layer reads are kept, with the same names, defaults,
derived values and validation; any object carrying these attributes (such as
the reference's own ModelConfig) can be passed to MoEGate / MoELayer. The ``router_*``
fields are this package's (the reference has one form of router, their defaults) and may be missing.
"""

from __future__ import annotations

import math
from dataclasses import dataclass, field


@dataclass
class ModelConfig:
    hidden_size: int = 512
    # fine-grained MoE: 32 routed + 2 shared experts, top-2 routed (model_config.py:53-58)
    intermediate_size: int = 160
    n_experts: int = 34
    n_shared_experts: int = 2
    n_experts_per_token: int = 2
    # the router's form (zmoe.functional.route)
    router_score: str = "sigmoid"      # or "softmax"
    router_bias: bool = True           # select by score + expert_biases
    router_groups: int = 1             # groups of experts, of which ...
    router_top_groups: int = 1         # ... so many are chosen from
    router_group_scores: int = 2       # a group's score: the sum of its 2 best experts' scores, or its best (1)
    router_renormalize: bool = True    # a token's weights sum to router_scale
    router_scale: float = 1.0
    n_routed_experts: int = field(init=False)
    initializer_range: float = field(init=False)

    def __post_init__(self):
        self.n_routed_experts = self.n_experts - self.n_shared_experts          # :135
        self.initializer_range = 1.0 / math.sqrt(self.hidden_size)              # :138
        if self.n_routed_experts <= 0:
            raise ValueError("n_experts must be greater than n_shared_experts.")
        if self.n_experts_per_token <= 0:
            raise ValueError("n_experts_per_token must be positive.")
        if self.n_experts_per_token > self.n_routed_experts:
            raise ValueError("n_experts_per_token cannot exceed n_routed_experts.")
        if self.router_score not in ("sigmoid", "softmax"):
            raise ValueError("router_score must be 'sigmoid' or 'softmax'.")
        groups = self.router_groups
        if groups < 1 or self.n_routed_experts % groups != 0:
            raise ValueError("router_groups must divide the routed experts.")
        if not 1 <= self.router_top_groups <= groups:
            raise ValueError("router_top_groups must be between 1 and router_groups.")
        if self.router_group_scores not in (1, 2) or (groups > 1 and self.router_group_scores > self.n_routed_experts // groups):
            raise ValueError("router_group_scores must be 1 or 2, and at most the experts of a group.")
        if self.n_experts_per_token > self.router_top_groups * (self.n_routed_experts // groups):
            raise ValueError("n_experts_per_token cannot exceed the experts of router_top_groups groups.")
