"""8-bit linear layers in a model, as far as the CPU goes."""
import torch
from torch import nn

from latest_exact_match_attention_amd import fp8
from latest_exact_match_attention_amd.model import ModelConfig, Transformer, load_trained


def held(lin: nn.Linear) -> fp8.Fp8Linear:
    n, k = lin.weight.shape
    kb = -(-k // 128)
    return fp8.Fp8Linear(fp8.Fp8(torch.zeros(n, kb * 128, dtype=torch.float8_e4m3fn),
                                 torch.ones(-(-n // 128), kb).to(torch.float8_e8m0fnu), k))


def test_parameter_counts():
    """A weight counts whichever way it is held."""
    m = Transformer(ModelConfig(vocab_size=256, depth=2, dim=96, num_heads=4))
    want, inner = m.n_params(), m.n_params(embedding=False)
    assert inner == want - 2 * 256 * 96
    m.blocks[0].mlp.up = held(m.blocks[0].mlp.up)
    assert (m.n_params(), m.n_params(embedding=False)) == (want, inner)
    m.lm_head = held(m.lm_head)
    assert (m.n_params(), m.n_params(embedding=False)) == (want, inner)


def test_a_checkpoint_loads(tmp_path):
    geo = dict(vocab_size=256, depth=2, dim=96, num_heads=4)
    m = Transformer(ModelConfig(**geo))
    m.blocks[1].mlp.down = held(m.blocks[1].mlp.down)
    m.blocks[1].mlp.down.values.random_(0, 100)
    m.lm_head = held(m.lm_head)
    torch.save({"config": geo, "state_dict": m.state_dict()}, tmp_path / "model.pt")
    got, _ = load_trained(tmp_path, device="cpu")
    assert type(got.blocks[1].mlp.down) is fp8.Fp8Linear and type(got.blocks[0].mlp.down) is nn.Linear
    for k, v in m.state_dict().items():
        assert torch.equal(got.state_dict()[k], v), k
