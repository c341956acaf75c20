"""Where the decoder's table of rotary frequencies lives: beside the module's own buffers, in float64, and never as a tensor of
inference mode (no GPU: the meta device stands for another one)."""
import pytest
import torch

from lucid_amd.modeling_lucid import LlamaRotaryEmbedding, LucidConfig

SCALED = dict(head_dim=64, rope_scaling={"rope_type": "linear", "factor": 4.0})


def _pass(emb, device):
    x = torch.empty(1, 3, 8, device=device)
    return emb(x, torch.zeros(1, 3, dtype=torch.int64, device=device))


@pytest.mark.parametrize("moved", [False, True], ids=["input elsewhere", "module moved"])
def test_a_first_pass_in_inference_mode_does_not_spoil_later_gradients(moved):
    """A tensor made in inference mode cannot be saved for a backward; the table is used by every later pass."""
    emb = LlamaRotaryEmbedding(LucidConfig(**SCALED))
    with torch.inference_mode():
        if moved:
            emb.to("meta")
        _pass(emb, "meta")
    assert not _pass(emb, "meta").inv_freq.is_inference()
    assert not _pass(emb, "cpu").inv_freq.is_inference()


def test_the_table_moves_with_the_module_and_stays_64_bits():
    """A pass finds the table where the module is (a captured one cannot copy it from the host)."""
    emb = LlamaRotaryEmbedding(LucidConfig(**SCALED))
    want = _pass(emb, "cpu").inv_freq.clone()
    emb.to(torch.bfloat16).to("meta")
    assert emb._placed.device.type == "meta" and emb._placed.dtype == torch.float64
    table = _pass(emb, "meta").inv_freq
    assert table is emb._placed
    back = emb.to_empty(device="cpu")  # (the values come from the host's table again)
    got = _pass(back, "cpu").inv_freq
    assert got.dtype == torch.float64 and torch.equal(got, want)


def test_default_positions_keep_their_buffer():
    emb = LlamaRotaryEmbedding(LucidConfig(head_dim=64)).to(torch.bfloat16)
    assert emb.inv_freq.dtype == torch.bfloat16 and len(_pass(emb, "cpu")) == 2
