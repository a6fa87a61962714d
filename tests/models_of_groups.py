"""An architecture whose layers route to experts in groups, as a user of the framework registers one: the feed-forward by its registered name,
its sizes where the builder looks for them."""

from types import SimpleNamespace

import beholdd
from beholdd.models import build_decoder

SIZES = SimpleNamespace(experts=16, top=3, expert_ff=48, shared_ff=56, groups=4, keep_groups=2, factor=2.5)


class GroupsConfig(beholdd.Qwen3Config):
    """Qwen3's layers with the feed-forward changed."""

    @property
    def layers(self):
        return [SimpleNamespace(mlp=SIZES)] * self.n_layers

    def layer_kinds(self):
        return [beholdd.LayerKinds(mixer=kinds.mixer, feed_forward="routed_experts_in_groups", norm=kinds.norm, block=kinds.block) for kinds in super().layer_kinds()]


CONFIG = {"architectures": ["ExpertsInGroups"], "num_hidden_layers": 3, "hidden_size": 128, "num_attention_heads": 4, "num_key_value_heads": 2, "head_dim": 32,
          "intermediate_size": 64, "vocab_size": 301, "rope_theta": 10000.0, "rms_norm_eps": 1e-5, "max_position_embeddings": 256, "tie_word_embeddings": False}


def folder(path, dtype="float32"):
    """A folder of random weights; the architecture is registered for as long as the process lasts, or `unregister` is called."""
    if "ExpertsInGroups" not in beholdd.registered_architectures():
        beholdd.register_architecture("ExpertsInGroups", GroupsConfig, build_decoder)
    beholdd.write_random_model(path, CONFIG, seed=4, dtype=dtype, std=0.1)
    return path


def unregister():
    beholdd.registry.unregister_architecture("ExpertsInGroups")
