"""What Umt5Encoder.encode_packed takes as prompts."""
import numpy as np
import pytest
import torch

from turbodiffusion_amd import text_encoder as TE

pytestmark = pytest.mark.gpu


def test_ids_of_any_whole_type_and_no_others():
    enc = TE.Umt5Encoder(TE.synthetic_state_dict(layers=1, dim=256, dim_ffn=512, heads=4, vocab=97, dtype=torch.float32))
    want = enc.encode_packed([torch.tensor([5, 6, 7]), torch.tensor([9])])
    for ps in ([[5, 6, 7], [9]], [np.array([5, 6, 7], np.int32), np.array([9])], [torch.tensor([5, 6, 7], dtype=torch.int32, device="cuda"), (9,)],
               [[5.0, 6.0, 7.0], torch.tensor([9.0])]):
        assert all(torch.equal(a, b) for a, b in zip(enc.encode_packed(ps), want))
    assert [t.shape[0] for t in enc.encode_packed([[], [9], []])] == [0, 1, 0] and enc.encode_packed([]) == []
    for bad in ([5, 6.5], torch.tensor([5.25], device="cuda"), [float("nan")], [float("inf")], [97], [-1]):
        with pytest.raises(ValueError):
            enc.encode_packed([[5], bad])
