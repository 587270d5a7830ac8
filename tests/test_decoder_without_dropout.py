'''Decoders unpickled from before `dropout` was among their attributes run without it.'''
import torch

from motif.model.config import MotifChordConfig
from motif.model.motif import MotifChordModel


def test_a_decoder_without_the_attribute():
    torch.manual_seed(0)
    model = MotifChordModel(MotifChordConfig(vocab_size=32, model_dim=64, num_heads=2, num_kv_heads=1, head_k_dim=32,
                                             block=('gdn', 'chord'), block_n=1))
    ids = torch.arange(7).view(1, 7)
    want = [model.train(mode)(ids).logits for mode in (True, False)]
    for block in model.blocks:
        for decoder in block.features:
            decoder.__dict__.pop('dropout')
    for mode, logits in zip((True, False), want):
        assert torch.equal(model.train(mode)(ids).logits, logits)
