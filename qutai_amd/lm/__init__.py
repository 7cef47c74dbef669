from .config import Config
from .decoder import Decoder
from .layers import GQA, Block, Projection, RMSNorm, SparseMoE, SwiGLU, attention_products, linear, projection_loss
from .layers import qk_norm_rope, rope, sample, silu_mul
from .packing import Packing
from .precision import autocast
from .rotary import Rotary
from .recompute import checkpoint as activation_checkpoint
from .checkpoint import checkpoint_metadata, load_checkpoint, load_weights, save_checkpoint, save_weights

__all__ = ["Block", "Config", "Decoder", "GQA", "Packing", "Projection", "RMSNorm", "Rotary", "SparseMoE", "SwiGLU", "activation_checkpoint",
           "attention_products", "autocast", "checkpoint_metadata", "linear", "load_checkpoint", "load_weights",
           "projection_loss", "qk_norm_rope", "rope", "sample", "save_checkpoint", "save_weights", "silu_mul"]
