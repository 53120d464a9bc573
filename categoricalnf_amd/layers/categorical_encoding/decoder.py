"""Embedding layer factory and the small decoder MLP (layers/categorical_encoding/decoder.py)."""
import torch
import torch.nn as nn
import torch.nn.functional as F

from ... import functional as Fn
from ...host_utils import get_param_val
from ..networks.help_layers import LinearNet

_NO_CLASS = -2 ** 63         # no category is left out: one outside the vocabulary is an error


def _hooked(module):
    """Whether a call of the module runs anything besides its forward()."""
    m = nn.modules.module
    return bool("forward" in module.__dict__ or module._forward_hooks or module._forward_pre_hooks or module._backward_hooks or module._backward_pre_hooks
                or m._global_forward_hooks or m._global_forward_pre_hooks or m._global_backward_hooks or m._global_backward_pre_hooks)


def create_embed_layer(vocab, vocab_size, default_embed_layer_dims):
    """nn.Embedding from scratch or from a torchtext vocabulary's vectors (decoder.py:12-21)."""
    use_vectors = (vocab is not None and vocab.vectors is not None)
    dims = vocab.vectors.shape[1] if use_vectors else default_embed_layer_dims
    vocab_size = len(vocab) if use_vectors else vocab_size
    embed = nn.Embedding(vocab_size, dims)
    if use_vectors:
        embed.weight.data.copy_(vocab.vectors)
        embed.weight.requires_grad = True
    return embed, vocab_size


def create_decoder(num_categories, num_dims, config, **kwargs):
    return DecoderLinear(num_categories, embed_dim=num_dims,
                         hidden_size=get_param_val(config, "hidden_size", 64),
                         num_layers=get_param_val(config, "num_layers", 1), **kwargs)


class DecoderLinear(nn.Module):
    """MLP latent -> class log-probabilities on the features [z, elu(z), elu(-z)] (decoder.py:35-63).
    The hidden layers are dense GEMMs of PyTorch-ROCm; `class_log_prob` ends in this package's linear cross entropy."""

    def __init__(self, num_categories, embed_dim, hidden_size, num_layers, class_prior_log=None):
        super().__init__()
        self.hidden_size = hidden_size
        self.num_layers = num_layers
        self.layers = LinearNet(c_in=3 * embed_dim, c_out=num_categories, num_layers=num_layers, hidden_size=hidden_size)
        self.log_softmax = nn.LogSoftmax(dim=-1)
        if class_prior_log is not None:
            if not isinstance(class_prior_log, torch.Tensor):
                class_prior_log = torch.from_numpy(class_prior_log)
            self.layers.set_bias(class_prior_log)

    def _features(self, z_cont):
        return torch.cat([z_cont, F.elu(z_cont), F.elu(-z_cont)], dim=-1)

    def forward(self, z_cont):
        return self.log_softmax(self.layers(self._features(z_cont)))

    def class_log_prob(self, z_cont, z_categ):
        """log p(z_categ | z_cont) for z_categ of z_cont's shape without its last axis: forward() gathered at one class, whose
        [..., C] log-probabilities are never written (one fused kernel per direction instead of GEMM + log-softmax + gather).  The kernel
        reads the last Linear's parameters and does not call the modules that it stands for: where one of them is hooked, replaced or
        watched, this is the gather."""
        net = self.layers.main_net
        last = net[-1] if type(net) is nn.Sequential else None
        if type(last) is not nn.Linear or type(self.log_softmax) is not nn.LogSoftmax or Fn.transformed() \
                or any(_hooked(m) for m in (self, self.layers, net, last, self.log_softmax)):
            scores = self(z_cont)
            inside = (z_categ >= 0) & (z_categ < scores.size(-1))        # outside: NaN, as the kernel's (an index error would end the process)
            chosen = scores.gather(-1, torch.where(inside, z_categ, 0).long().unsqueeze(-1)).squeeze(-1)
            return torch.where(inside, chosen, float("nan"))
        hidden = self.layers.hidden_features(self._features(z_cont)).to(last.weight.dtype)          # autocast: back from 16 bits
        return -Fn.linear_cross_entropy(hidden, last.weight, z_categ, last.bias, ignore_index=_NO_CLASS, reduction="none")

    def info(self):
        return "Linear model with hidden size %i and %i layers" % (self.hidden_size, self.num_layers)
