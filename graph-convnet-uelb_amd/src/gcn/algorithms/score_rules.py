"""Rules on link scores ``[B, V, V, C]`` before paths are drawn from them or searched in them: links without capacity are masked,
links that earlier paths use are penalised, and a bias and a temperature can be applied.  The result goes where the scores
went: ``PathSampler``, ``BeamSearchFactory`` and the losses on it.  Differentiable in the scores and in the bias.

Every row (graph b, node i, commodity c) is a distribution over the next node j; its history is the hops that the given paths make
from node i in graph b, whatever their commodity.  The reference has no counterpart (its sampler draws the commodities
independently, ``src/gcn/algorithms/path_sampler.py:51-214``).
"""
from __future__ import annotations

import torch

from ..hip import lib as L
from ..hip.logits import pack_mask, process_logits


def hops_from(paths, path_len, num_nodes):
    """``[B, V, N]``: for every node the next node on each of N paths, -1 where a path does not leave it.  paths ``[B, N, PL]``
    (padded with anything behind path_len ``[B, N]``); a path visits a node once."""
    B, N, PL = paths.shape
    paths = paths.long()
    here, there = paths[:, :, :-1], paths[:, :, 1:]
    inside = torch.arange(1, PL, device=paths.device) < path_len.unsqueeze(-1)
    inside &= (here >= 0) & (here < num_nodes) & (there >= 0) & (there < num_nodes)
    # hops outside go to a row of their own that is cut off
    hops = torch.full((B, num_nodes + 1, N), -1, dtype=torch.int32, device=paths.device)
    place = torch.where(inside, here, num_nodes).transpose(1, 2)                      # [B, PL - 1, N]
    hops.scatter_(1, place, torch.where(inside, there, -1).transpose(1, 2).to(torch.int32))
    return hops[:, :num_nodes].contiguous()


class LinkScoreRules:
    """edges_capacity ``[B, V, V]``: links without capacity and self loops are masked (masked_value).  repetition_penalty,
    presence_penalty, frequency_penalty: for links that the paths of a call use; temperature, bias (float32 ``[V]``, ``[V, V]`` or
    ``[B, V, V]``): see ``process_logits``."""

    def __init__(self, edges_capacity, repetition_penalty=1.0, presence_penalty=0.0, frequency_penalty=0.0, bias=None, temperature=1.0,
                 masked_value=-1e9):
        L.require_cuda(edges_capacity, "edges_capacity")
        if edges_capacity.dim() != 3 or edges_capacity.shape[1] != edges_capacity.shape[2]:
            raise ValueError(f"edges_capacity must be [batch, nodes, nodes], got {tuple(edges_capacity.shape)}")
        self.batch_size, self.num_nodes = edges_capacity.shape[:2]
        loops = torch.eye(self.num_nodes, dtype=torch.bool, device=edges_capacity.device)
        self.mask = pack_mask((edges_capacity > 0) & ~loops)
        self.bias, self.masked_value = bias, masked_value
        self.kind = dict(repetition_penalty=repetition_penalty, presence_penalty=presence_penalty, frequency_penalty=frequency_penalty,
                         temperature=temperature)

    def __call__(self, scores, paths=None, path_len=None):
        """The scores after the rules; paths ``[B, N, PL]`` / path_len ``[B, N]`` are those whose links are penalised."""
        if scores.dim() != 4 or scores.shape[:3] != (self.batch_size, self.num_nodes, self.num_nodes):
            raise ValueError(f"scores must be [{self.batch_size}, {self.num_nodes}, {self.num_nodes}, commodities], got {tuple(scores.shape)}")
        if (paths is None) != (path_len is None):
            raise ValueError("paths and path_len go together")
        history = None
        if paths is not None:
            if paths.dim() != 3 or paths.shape[0] != self.batch_size or path_len.shape != paths.shape[:2]:
                raise ValueError("paths must be [batch, paths, length] and path_len [batch, paths]")
            history = hops_from(paths, path_len, self.num_nodes)
        return process_logits(scores, dim=2, history=history, bias=self.bias, mask=self.mask, masked_value=self.masked_value, **self.kind)
