"""The MLP bodies of the VAEs (model/spherical_vae.py:30-66, 85-101: Linear + softplus), and their form for wide layers and
large batches.  Two optional config keys; without them the bodies are the stock ones.

  config["hidden"] = "blocks8"   the hidden layers and the decoder's output layer multiply in 8-bit blocks, and each keeps
                                 one byte per activation for the backward pass (blocks8.linear).  The layers at the data,
                                 at the latent variable and the posterior heads stay as they are.
  config["layer_norm"] = True    a layer norm in front of every softplus (norm.LayerNorm; modules encoder_norms and
                                 decoder_norms)

Against softplus + nn.Linear the 8-bit layer (forward and gradients) was no slower at any size measured; what it gains grows
with rows times width.  fp32, captured in a graph: 128 x 128 x 128 (rows, in, out) 29 us for 43, 1024 x 1024 x 1024 53 for 88,
16384 x 128 x 784 80 for 217, 16384 x 2048 x 2048 0.68 ms for 2.98; a call by itself at batch 128 is the Python's time either
way (142 us for 156).  What it costs is the operands' 3 bits of mantissa.  It keeps a byte for every element of its input where
float32 keeps eight (the activation and what softplus needs), and a byte for every element of the weight: with fewer rows than
columns that can be more (1024 x 4096 x 4096: 21 MB for 17).

The models train in float32: the 8-bit layer and the norm also take float16 and bfloat16, the posterior samplers do not, so
under torch.autocast the heads' outputs have to be cast before they are sampled; the 16-bit forms are for callers of
blocks8.linear and norm.layer_norm.  In float64 the norm runs and the 8-bit layer refuses.
"""
from collections.abc import Mapping

import torch.nn as nn
import torch.nn.functional as F

from .. import blocks8
from ..norm import LayerNorm


def _option(config, key, default):
    if isinstance(config, Mapping) and key not in config:  # (a defaultdict would invent a value)
        return default
    try:
        return config[key]
    except KeyError:
        return default


def prepare(model):
    """reads the two keys of model.config and adds the norms; called at the end of a model's constructor"""
    config = model.config
    hidden = _option(config, "hidden", None)
    if hidden not in (None, "blocks8"):
        raise ValueError(f"config['hidden'] must be absent, None or 'blocks8', got {hidden!r}")
    model._hidden_kind = hidden
    if _option(config, "layer_norm", False):
        for side in ("encoder", "decoder"):
            setattr(model, side + "_norms", nn.ModuleList(
                [LayerNorm(config[side + "_width"], device=model.device) for _ in range(config[side + "_depth"] + 1)]))


def _linear(model, layer, h):
    """layer(softplus(h))"""
    if getattr(model, "_hidden_kind", None) == "blocks8":  # (a model pickled without the attribute is a stock one)
        return blocks8.linear(h, layer.weight, layer.bias, "softplus", model.sftbeta)
    return layer(F.softplus(h, beta=model.sftbeta))


def _before_last_softplus(model, side, x):
    h = getattr(model, side + "_function")(x)
    norms = getattr(model, side + "_norms", None)
    if norms is not None:
        h = norms[0](h)
    for i, layer in enumerate(getattr(model, side + "_linear_layers")):
        h = _linear(model, layer, h)
        if norms is not None:
            h = norms[i + 1](h)
    return h


def encode(model, x):
    """the encoder's last hidden activation, which the heads read"""
    return F.softplus(_before_last_softplus(model, "encoder", x), beta=model.sftbeta)


def decode(model, z):
    return _linear(model, model.function_x_mu, _before_last_softplus(model, "decoder", z))
