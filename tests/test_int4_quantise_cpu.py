"""LlamaForCausalLM.quantize_weights_int4 that is refused or interrupted, on the CPU: the
quantiser runs, the packing kernel is left out."""
import pytest
import torch

from llama_pure_compute_b200 import int4_linear
from llama_pure_compute_b200.config import LlamaModelConfig
from llama_pure_compute_b200.model import LlamaForCausalLM

SMALL = dict(vocab_size=64, dim=128, inter_dim=192, num_layers=3, num_heads=2, num_kv_heads=1,
             max_seq_len=32)


@pytest.fixture
def packed(monkeypatch):
    """Names of the weights that were packed; `packed.room`: how many more fit."""
    class Packed(list):
        room = 99

    done = Packed()

    def pack(self, codes, scales, mins, layout, group_size):
        if not done.room:
            raise torch.OutOfMemoryError("no room")
        done.room -= 1
        done.append(tuple(codes.shape))
    monkeypatch.setattr(int4_linear, "_require_cuda", lambda t, n: None)
    monkeypatch.setattr(int4_linear.Int4Weight, "_pack", pack)
    return done


def build():
    torch.manual_seed(0)
    return LlamaForCausalLM(LlamaModelConfig(**SMALL)).to(torch.bfloat16)


def state(model):
    return {n: t.clone() for n, t in model.state_dict().items()}


def untouched(model, before):
    now = model.state_dict()
    return now.keys() == before.keys() and all(
        torch.equal(now[n].nan_to_num(nan=-9.0, posinf=9e9), t.nan_to_num(nan=-9.0, posinf=9e9))
        for n, t in before.items())


@pytest.mark.parametrize("where", ["down_proj", "lm_head", "o_proj"])
@pytest.mark.parametrize("bad", ["nan", "range", "type"])
def test_a_refused_weight_leaves_the_model_as_it_was(packed, where, bad):
    model = build()
    last = model.model.layers[-1]
    lin = {"down_proj": last.down_proj, "lm_head": model.lm_head, "o_proj": last.self_attn.o_proj}[where]
    good = lin.weight.detach().clone()
    if bad == "nan":
        lin.weight.data[3, 5] = float("nan")
    elif bad == "range":
        lin.weight.data[3, :2] = torch.tensor([3e38, -3e38])
    else:
        lin.weight.data = lin.weight.data.float()
    before = state(model)
    with pytest.raises(TypeError if bad == "type" else ValueError, match="LlamaPureComputeError"):
        model.quantize_weights_int4(64)
    assert untouched(model, before) and not packed
    assert model.model.layers[0].int4_down is None and model.int4_lm_head is None
    lin.weight.data = good
    model.quantize_weights_int4(64)
    assert len(packed) == 3 * 4 + 1


@pytest.mark.parametrize("room", range(13))
def test_running_out_of_memory_can_be_gone_on_from(packed, room):
    """Every weight is either whole in 16 bits or in 4 at each point, and a second call
    finishes."""
    model = build()
    packed.room = room
    with pytest.raises(torch.OutOfMemoryError):
        model.quantize_weights_int4(64)
    for layer in model.model.layers:
        a = layer.self_attn
        for lin, four in ((a.q_proj, a.int4_qkv), (a.o_proj, a.int4_o), (layer.up_proj, layer.int4_gate_up),
                          (layer.down_proj, layer.int4_down)):
            assert (lin.weight.shape[0] == 0) == (four is not None)
    packed.room = 99
    model.quantize_weights_int4(64)
    assert model.int4_lm_head is not None and model.lm_head.weight.shape[0] == 0
    assert all(layer.down_proj.weight.shape[0] == 0 for layer in model.model.layers)
    with pytest.raises(RuntimeError, match="already"):
        model.quantize_weights_int4(64)


def test_the_vocabulary_projection_can_follow_later(packed):
    model = build()
    model.quantize_weights_int4(64, lm_head=False)
    assert model.int4_lm_head is None and len(packed) == 12
    with pytest.raises(RuntimeError, match="already"):
        model.quantize_weights_int4(64, lm_head=False)
    model.quantize_weights_int4(64)
    assert len(packed) == 13 and model.int4_lm_head is not None
