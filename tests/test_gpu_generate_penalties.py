"""ScopeDecoder.generate with penalties that are refused, and with positions past 32 bits."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_refused_penalties_leave_the_decoder_where_it_was():
    from scope_amd.decode import DecoderConfig, ScopeDecoder

    cfg = DecoderConfig(vocab_size=1000, num_layers=6, num_heads=2, model_dim=256, no_attn_layer=3)
    prompt = torch.randint(0, 1000, (256,), generator=torch.Generator().manual_seed(3)).to(DEV)
    m = ScopeDecoder(cfg, max_len=512, seed=1)
    first = int(m.prefill(prompt)[:1000].argmax())
    for bad, error in ((dict(repetition=0.0), ValueError), (dict(temperature=1e-50), ValueError), (dict(bias=torch.zeros(999, device=DEV)), RuntimeError),
                       (dict(mask=torch.zeros(32, dtype=torch.int64, device=DEV)), RuntimeError), (dict(wrong=1), TypeError),
                       (dict(out=torch.zeros(1000, device=DEV)), TypeError)):
        with pytest.raises(error):
            m.generate(3, first, penalties=bad)
        assert m.t == 256 and int(m._t_dev) == 256
    # nothing counts from there on, and nothing is in a history that starts there: as without penalties
    want = m.generate(5, first).tolist()
    for none in (dict(n_prompt=2 ** 40, frequency=5.0, presence=5.0), dict(first=2 ** 63 - 1, repetition=9.0, frequency=5.0)):
        m.prefill(prompt)
        assert m.generate(5, first, penalties=none).tolist() == want
