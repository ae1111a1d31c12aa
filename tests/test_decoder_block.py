"""The decoder block with a token mixer of the caller's own (no GPU)."""

import torch
from torch import nn


class Scale(nn.Module):
    """A mixer with the plainest signature: x -> (output, cache)."""

    def forward(self, x):
        return 2 * x, None


def test_block_calls_a_plain_mixer():
    from nlogn_pisa_b200.model import BlockConfig, DecoderBlock

    block = DecoderBlock(BlockConfig(vocab_size=50, hidden_size=64, intermediate_size=96, num_attention_heads=2,
                                     num_key_value_heads=1, head_dim=32))
    block.attn = Scale()
    tokens = torch.randint(0, 50, (2, 7))
    x = block.embed(tokens)
    x = x + 2 * block.norm1(x)
    assert torch.equal(block(tokens), block.norm_out(x + block.ffn(block.norm2(x))))
