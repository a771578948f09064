"""The block says which of its options are in effect."""
import torch


def test_mxfp4_weights_have_no_fused_epilogues(pkg):
    params = {"w4_qkv": torch.zeros(1), "heads": 2, "head_dim": 128, "ffn": 512}
    block = pkg.block.DiTBlock(params)
    assert block.mxfp4 and block.fuse_residual is False and block.fuse_swiglu is False
    int8 = {"heads": 2, "head_dim": 128, "ffn": 100}         # ffn is no multiple of the interleaving
    assert pkg.block.DiTBlock(int8).fuse_residual is True and pkg.block.DiTBlock(int8).fuse_swiglu is False
    assert pkg.block.DiTBlock(int8, fuse_residual=False).fuse_residual is False
