"""The Kogarashi layer refuses tensors that its kernels would decode with other sizes or types than they have, before any address
reaches the library. No GPU: descriptors of layers whose tensors lie in host memory, none of which is ever launched."""
import pytest
import torch

H, I, E = 512, 256, 4


def layer(**changes):
    """A layer as `load` leaves it (Q6_K regrouped), with tensors replaced: name=(type, ne) or name=(type, ne, bytes)."""
    import darask_inference_engine_b200 as D
    from darask_inference_engine_b200 import formats as F
    m = object.__new__(D.KogarashiMoeLayer)
    m.hidden, m.inter, m.experts, m.topk, m.max_tokens = H, I, E, 2, 4
    m.router_bias, m.workspace = None, torch.zeros(16, dtype=torch.uint8)
    m.weights = D.kogarashi._Tensors()
    tensors = dict(gate_inp=(0, (H, E)), gate_exps=(12, (H, I, E)), up_exps=(12, (H, I, E)), down_exps=(14, (I, H, E)), gate_shexp=(12, (H, I)),
                   up_shexp=(12, (H, I)), down_shexp=(14, (I, H)), gate_inp_shexp=(0, (H,)))
    tensors.update(changes)
    for name, spec in tensors.items():
        if spec is None:
            continue
        ty, ne = spec[:2]
        rows = 1
        for d in ne[1:]:
            rows *= d
        nbytes = spec[2] if len(spec) > 2 else rows * F.q6k_r16_row_bytes(ne[0]) if ty == 14 else F.ggml_tensor_bytes(ty, ne)
        m.weights[f"ffn_{name}.weight"] = D.kogarashi.Weight(torch.zeros(nbytes, dtype=torch.uint8), ty, ne[0], ne[1] if len(ne) > 1 else 1, tuple(ne))
    return m


def descriptor(m):
    x = torch.zeros(2, H)
    return m._descriptor(x, x.clone(), None, None, 1e-6)


@pytest.mark.parametrize("good", [dict(), dict(gate_shexp=None, up_shexp=None, down_shexp=None, gate_inp_shexp=None), dict(gate_inp_shexp=(0, (H, 1))),
                                  dict(down_exps=(12, (I, H, E)), down_shexp=(12, (I, H))), dict(gate_inp=(30, (H, E)), gate_inp_shexp=(30, (H,))),
                                  dict(gate_exps=(14, (H, I, E)), up_exps=(14, (H, I, E)), gate_shexp=(14, (H, I)), up_shexp=(14, (H, I)))])
def test_a_layer_whose_tensors_fit_passes(good):
    m = layer(**good)
    d = descriptor(m)
    assert d.gate_w == m.weights["ffn_gate_exps.weight"].data.data_ptr()
    assert (d.sh_down_w is None) == ("gate_shexp" in good and good["gate_shexp"] is None)


@pytest.mark.parametrize("bad", [
    dict(down_shexp=(12, (I, H))),                                     # a shared down of another type than the routed ones
    dict(down_exps=(12, (I, H, E))),
    dict(gate_shexp=(14, (H, I)), up_shexp=(14, (H, I))), dict(up_shexp=(14, (H, I))), dict(up_exps=(14, (H, I, E))),
    dict(gate_inp_shexp=(30, (H,))), dict(gate_inp=(1, (H, E))),       # a shared gate of another type than the router
    dict(gate_shexp=(12, (H, I // 2))), dict(down_shexp=(14, (I * 2, H))),      # a shared expert of another width
    dict(gate_shexp=(12, (H, I, 2))), dict(gate_exps=(12, (H, I, E - 1))), dict(up_exps=(12, (H, I))), dict(down_exps=(14, (I, H // 2, E))),
    dict(gate_inp=(0, (H, E + 1))), dict(gate_inp=(0, (H // 2, E))), dict(gate_inp_shexp=(0, (H // 2,))),
    dict(gate_exps=(0, (H, I, E))), dict(gate_inp=(12, (H, E))),
    dict(gate_exps=(12, (H, I, E), 144)), dict(down_exps=(14, (I, H, E), E * H * 210)),      # fewer bytes; Q6_K that was not regrouped
], ids=str)
def test_tensors_that_do_not_fit_are_refused(bad):
    with pytest.raises(ValueError, match="|".join(f"ffn_{n}" for n in ("gate", "up", "down"))):
        descriptor(layer(**bad))


def test_tensors_replaced_later_are_looked_at_again():
    import darask_inference_engine_b200 as D
    m = layer()
    descriptor(m)
    w = m.weights["ffn_down_shexp.weight"]
    m.weights["ffn_down_shexp.weight"] = D.kogarashi.Weight(w.data[:-16], w.ty, w.k, w.rows, w.ne)
    for _ in range(2):                                                 # and again until it is put right
        with pytest.raises(ValueError, match="ffn_down_shexp"):
            descriptor(m)
    m.weights.update({"ffn_down_shexp.weight": w})
    descriptor(m)


def test_strided_inputs_of_the_layer_entry_are_refused():
    """The entry kernel reads attn_out and norm_w as packed rows: views with strides gave other numbers."""
    m = layer()
    x, norm = torch.zeros(2, H), torch.ones(H)
    for attn_out, norm_w in ((torch.zeros(2, 2 * H)[:, :H], norm), (torch.zeros(H, 2).t(), norm), (x.clone(), torch.ones(2 * H)[::2]), (None, torch.ones(2 * H)[::2])):
        with pytest.raises(ValueError, match="norm_w"):
            m._descriptor(x, x.clone(), attn_out, norm_w, 1e-6)
    d = m._descriptor(x, x.clone(), x, norm, 1e-6)
    assert d.attn_out == x.data_ptr() and d.norm_w == norm.data_ptr()
