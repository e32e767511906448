"""Import of FP8 checkpoints: what a checkpoint keeps out of the quantisation (sensitive projections, the embedding, the head) comes out in its own 16 or 32 bits."""
import json
import os

import numpy as np
import pytest
import torch

from machx_inference_engine_b200.formats.gguf import GGMLType, GGUFReader
from machx_inference_engine_b200.formats.hf_import import import_to_gguf
from machx_inference_engine_b200.formats.safetensors import SafetensorsModel, write_safetensors
from machx_inference_engine_b200.models.sources import GGUFSource
from machx_inference_engine_b200.ops.weights import WFormat
from machx_inference_engine_b200.runtime.api import Engine
from machx_inference_engine_b200.runtime.engine import EngineOptions, SamplingParams
from test_fp8_models import hf_directory


def of_type(d, dtype, names):
    """Writes the directory's unquantised matrices of these names again, as ``dtype``."""
    st = SafetensorsModel(d)
    tensors = {n: ("F8_E4M3", st.numpy(n).copy()) if st.dtype(n) == "F8_E4M3" else st.numpy(n).copy() for n in st.names()}
    for n in tensors:
        if any(k in n for k in names) and st.dtype(n) != "F8_E4M3":
            v = torch.from_numpy(st.float32(n).copy())
            tensors[n] = ("BF16", v.to(torch.bfloat16).view(torch.int16).numpy().view(np.uint16)) if dtype == "BF16" else v.numpy().astype(np.float32 if dtype == "F32" else np.float16)
    del st
    write_safetensors(os.path.join(d, "model.safetensors"), tensors)


@pytest.mark.parametrize("dtype", ["F16", "BF16", "F32"])
def test_unquantised_matrices_are_kept(tmp_path, dtype):
    d = str(tmp_path)
    hf_directory(d, kept=("q_proj", "down_proj"))
    names = ("embed_tokens", "lm_head", "q_proj", "down_proj")
    of_type(d, dtype, names)
    st = SafetensorsModel(d)
    out = os.path.join(d, "out.gguf")
    import_to_gguf(d, out, log=lambda s: None)
    r = GGUFReader(out)
    src = GGUFSource(r, "cpu")
    want = {"F16": GGMLType.F16, "BF16": GGMLType.BF16, "F32": GGMLType.F32}[dtype]
    for hf, gg in (("model.embed_tokens.weight", "token_embd.weight"), ("lm_head.weight", "output.weight"), ("model.layers.1.mlp.down_proj.weight", "blk.1.ffn_down.weight"),
                   ("model.layers.0.self_attn.q_proj.weight", "blk.0.attn_q.weight")):
        v = torch.from_numpy(st.float32(hf).copy())
        assert st.dtype(hf) == dtype and r.tensor(gg).type == want
        stored = torch.from_numpy(r.tensor(gg).to_float32().reshape(v.shape).copy())
        if "q_proj" in hf:                                   # (the row order of llama files)
            v = v.reshape(4, 2, 32, -1).transpose(1, 2).reshape(v.shape)
        assert torch.equal(stored, v)
        w = src.matrix(gg, *v.shape)
        assert w.fmt == WFormat.BF16 and torch.equal(w.dequantize()[0], v.to(torch.bfloat16).float())
    assert r.tensor("blk.0.ffn_up.weight").type == GGMLType.I8
    eng = Engine.load(out, "cpu", EngineOptions(max_ctx=256, max_seqs=1))
    assert eng.generate("hello", SamplingParams(max_tokens=4, temperature=0.0)).completion_tokens >= 1


def test_a_matrix_in_64_bits_is_kept_in_32(tmp_path):
    d = str(tmp_path)
    hf_directory(d)
    st = SafetensorsModel(d)
    tensors = {n: ("F8_E4M3", st.numpy(n).copy()) if st.dtype(n) == "F8_E4M3" else st.numpy(n).copy() for n in st.names()}
    del st
    tensors["lm_head.weight"] = tensors["lm_head.weight"].astype(np.float64)
    write_safetensors(os.path.join(d, "model.safetensors"), tensors)
    import_to_gguf(d, os.path.join(d, "out.gguf"), log=lambda s: None)
    t = GGUFReader(os.path.join(d, "out.gguf")).tensor("output.weight")
    assert t.type == GGMLType.F32 and np.array_equal(t.to_float32().reshape(-1), tensors["lm_head.weight"].astype(np.float32).reshape(-1))


def test_checkpoints_of_other_kinds_are_imported_as_before(tmp_path):
    """Without a quantisation of their own, projections become Q4_K and the head Q6_K."""
    d = str(tmp_path)
    hf_directory(d, kept=("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj"))
    path = os.path.join(d, "config.json")
    cfg = json.load(open(path))
    del cfg["quantization_config"]
    json.dump(cfg, open(path, "w"))
    out = os.path.join(d, "out.gguf")
    import_to_gguf(d, out, log=lambda s: None)
    r = GGUFReader(out)
    assert r.tensor("blk.0.attn_v.weight").type == GGMLType.Q4_K and r.tensor("output.weight").type == GGMLType.Q6_K
