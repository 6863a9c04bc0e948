"""Gates that were pickled whole before they had a form: they are the reference's."""

import copy
import pickle

import torch


def test_a_gate_without_a_form():
    from modeling.model_config import ModelConfig
    from modeling.moe_gate import MoEGate

    config = ModelConfig(hidden_size=32, intermediate_size=16, n_experts=9, n_shared_experts=1, n_experts_per_token=2)
    gate = MoEGate(config)
    old = copy.deepcopy(gate)
    del old.__dict__["form"]
    for name in [n for n in vars(old.config) if n.startswith("router_")]:
        delattr(old.config, name)
    again = pickle.loads(pickle.dumps(old))
    assert again.form is None and again.score == "sigmoid" and torch.equal(again.weight, gate.weight)
    other = MoEGate(ModelConfig(hidden_size=32, intermediate_size=16, n_experts=9, n_shared_experts=1, n_experts_per_token=2,
                                router_score="softmax"))
    assert pickle.loads(pickle.dumps(other)).form == other.form and other.score == "softmax"
