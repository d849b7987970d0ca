"""Calls of the operators of strassen_hip/block.py that are easy to get wrong around their kernels: together with the other features of
the framework, on memory that is shared, under torch's transforms and hooks.  What needs no GPU runs without one."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import block_reference as ref


def _randn(shape, dtype, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype)


# ------------------------------------------------------------------------------------------ the swap of Linear layers
def test_swap_of_linear_layers_keeps_epilogues():
    """A LinearAct has an activation and takes a residual, which no Strassen layer has: it stays what it is."""
    from model.layers import LinearAct, LinearStrassen, LinearStrassenRect, replace_linear_with_strassen
    import torch.nn as nn
    layers = lambda: nn.ModuleDict({"act": LinearAct(256, 256, activation="silu", device="cpu"), "wide": LinearAct(256, 512, activation="gelu", device="cpu"),
                                    "plain": LinearAct(256, 256, device="cpu"), "inner": nn.Sequential(LinearAct(128, 128, activation="relu", device="cpu"), nn.Linear(128, 128))})
    for square_only in (True, False):
        m = layers()
        acts = [m["act"], m["wide"], m["plain"], m["inner"][0]]
        replace_linear_with_strassen(m, square_only=square_only)
        assert [m["act"], m["wide"], m["plain"], m["inner"][0]] == acts
        assert type(m["inner"][1]) is (LinearStrassen if square_only else LinearStrassenRect)


@pytest.mark.gpu
def test_fused_block_after_the_swap():
    """gpt_block_demo's FusedBlock gives the same bits before and after the swap of its Linear layers."""
    import gpt_block_demo as demo
    from model.layers import replace_linear_with_strassen
    torch.manual_seed(0)
    for square_only in (True, False):
        block = demo.FusedBlock(demo.Block(256, 4, dtype=torch.bfloat16, rotary=True))
        x = _randn((2, 70, 256), torch.bfloat16, 1).cuda()
        with torch.no_grad():
            before = block(x)
            replace_linear_with_strassen(block, square_only=square_only)
            assert torch.equal(block(x), before)
