"""FP8 checkpoints from file to tokens: synthetic GGUF files, import of a Hugging Face directory, dense and expert graphs on the CPU and the GPU, refusals."""
import json
import os

import numpy as np
import pytest
import torch

from machx_inference_engine_b200.formats.gguf import GGMLType, GGUFReader
from machx_inference_engine_b200.formats.hf_import import ImportError_, import_to_gguf, parse_hf_config
from machx_inference_engine_b200.formats.model_config import preset
from machx_inference_engine_b200.formats.safetensors import SafetensorsModel, write_safetensors
from machx_inference_engine_b200.formats.synth import write_synthetic_gguf
from machx_inference_engine_b200.models import build_model
from machx_inference_engine_b200.models.sources import GGUFSource
from machx_inference_engine_b200.ops.weights import WFormat, from_fp8
from machx_inference_engine_b200.runtime.api import Engine
from machx_inference_engine_b200.runtime.engine import EngineOptions, LLMEngine, SamplingParams


@pytest.mark.parametrize("name", ["tiny-llama", "tiny-qwen3moe", "tiny-qwen3next"])
def test_a_synthetic_file_loads_and_generates(tmp_path, name):
    path = str(tmp_path / "m.gguf")
    write_synthetic_gguf(preset(name), path, quant="fp8", seed=1)
    r = GGUFReader(path)
    assert r.tensor("blk.0.attn_output.weight" if name != "tiny-qwen3next" else "blk.0.ssm_out.weight").type == GGMLType.I8
    assert r.tensor("token_embd.weight").type == GGMLType.BF16
    eng = Engine.load(path, "cpu", EngineOptions(max_ctx=512, max_seqs=2))
    a = eng.generate("Hello world, the answer is", SamplingParams(max_tokens=5, temperature=0.0))
    b = eng.generate("Hello world, the answer is", SamplingParams(max_tokens=5, temperature=0.0))
    assert a.completion_tokens >= 1 and a.token_ids == b.token_ids


def test_matrices_and_experts_of_a_file(tmp_path):
    cfg = preset("tiny-qwen3moe")
    path = str(tmp_path / "m.gguf")
    write_synthetic_gguf(cfg, path, quant="fp8", seed=3)
    src = GGUFSource(GGUFReader(path), "cpu")
    bank = src.matrix("blk.0.ffn_up_exps.weight", cfg.expert_ffn, cfg.hidden, cfg.n_experts)
    assert bank.fmt == WFormat.FP8 and bank.E == cfg.n_experts
    share = src.matrix("blk.0.ffn_up_exps.weight", cfg.expert_ffn, cfg.hidden, cfg.n_experts, experts=(1, 3))
    assert torch.equal(share.dequantize(), bank.dequantize()[1:3])
    assert abs(float(bank.dequantize().std()) / 0.02 - 1) < 0.1
    with pytest.raises(ValueError):
        src.matrix("blk.0.ffn_up_exps.weight", cfg.expert_ffn + 1, cfg.hidden, cfg.n_experts)


def hf_directory(d, block=(128, 128), scheme="dynamic", kept=()):
    rng = np.random.default_rng(0)
    H, F, L, V, nh, nkv, hd = 256, 384, 2, 320, 4, 2, 64
    json.dump({"model_type": "llama", "architectures": ["LlamaForCausalLM"], "hidden_size": H, "intermediate_size": F, "num_hidden_layers": L, "num_attention_heads": nh,
               "num_key_value_heads": nkv, "head_dim": hd, "vocab_size": V, "max_position_embeddings": 512, "rms_norm_eps": 1e-6, "rope_theta": 10000.0,
               "quantization_config": {"quant_method": "fp8", "activation_scheme": scheme, "weight_block_size": list(block) if block else None}},
              open(os.path.join(d, "config.json"), "w"))
    tensors, dense = {}, {}

    def lin(name, n, k):
        if name.split(".")[-1] in kept:                      # a matrix that was left out of the quantisation
            w = rng.standard_normal((n, k)).astype(np.float16) * np.float16(0.02)
            tensors[name + ".weight"], dense[name] = w, torch.from_numpy(w.astype(np.float32))
            return
        codes = (torch.from_numpy(rng.standard_normal((n, k))).clamp(-4, 4) * 112).to(torch.float8_e4m3fn)
        s = (rng.random((-(-n // 128), -(-k // 128))).astype(np.float32) + 0.5) * np.float32(0.02 / 112)
        tensors[name + ".weight"] = ("F8_E4M3", codes.view(torch.uint8).numpy())
        tensors[name + ".weight_scale_inv"] = s
        dense[name] = from_fp8(codes, torch.from_numpy(s)).dequantize()[0]

    for i in range(L):
        p = f"model.layers.{i}."
        for name, n, k in (("self_attn.q_proj", nh * hd, H), ("self_attn.k_proj", nkv * hd, H), ("self_attn.v_proj", nkv * hd, H), ("self_attn.o_proj", H, nh * hd),
                           ("mlp.gate_proj", F, H), ("mlp.up_proj", F, H), ("mlp.down_proj", H, F)):
            lin(p + name, n, k)
        for n in ("input_layernorm", "post_attention_layernorm"):
            tensors[p + n + ".weight"] = np.ones(H, dtype=np.float16)
    tensors["model.embed_tokens.weight"] = (rng.standard_normal((V, H)) * 0.02).astype(np.float16)
    tensors["lm_head.weight"] = (rng.standard_normal((V, H)) * 0.02).astype(np.float16)
    tensors["model.norm.weight"] = np.ones(H, dtype=np.float16)
    write_safetensors(os.path.join(d, "model.safetensors"), tensors)
    from machx_inference_engine_b200.formats.synth import gpt2_byte_map
    json.dump({"model": {"type": "BPE", "vocab": {ch: i for i, ch in enumerate(gpt2_byte_map())}, "merges": []}, "added_tokens": []}, open(os.path.join(d, "tokenizer.json"), "w"))
    return dense


def test_import_keeps_the_codes(tmp_path):
    dense = hf_directory(str(tmp_path))
    st = SafetensorsModel(str(tmp_path))
    assert st.dtype("model.layers.0.mlp.up_proj.weight") == "F8_E4M3" and np.abs(st.float32("model.layers.0.mlp.up_proj.weight")).max() <= 448
    out = str(tmp_path / "out.gguf")
    import_to_gguf(str(tmp_path), out, log=lambda s: None)
    src = GGUFSource(GGUFReader(out), "cpu")
    for i, (hf, gg) in enumerate((("self_attn.q_proj", "attn_q"), ("mlp.down_proj", "ffn_down"))):
        want = dense[f"model.layers.{i}.{hf}"]
        w = src.matrix(f"blk.{i}.{gg}.weight", *want.shape)
        assert w.fmt == WFormat.FP8 and torch.equal(w.dequantize()[0], want)
    eng = Engine.load(out, "cpu", EngineOptions(max_ctx=256, max_seqs=1))
    q = eng.model.layers[0]["attn"].qkv.w                    # rows in the Hugging Face order: rotated in halves as they are
    assert torch.equal(q.dequantize()[0][:256], dense["model.layers.0.self_attn.q_proj"])
    assert eng.generate("hello", SamplingParams(max_tokens=4, temperature=0.0)).completion_tokens >= 1


@pytest.mark.parametrize("kept", ["q_proj", "k_proj"])
def test_queries_and_keys_of_two_kinds_keep_one_row_order(tmp_path, kept):
    """The matrices that a file stores without quantisation are in the interleaved order of llama files, the e4m3 ones in halves: each is read as what it is."""
    dense = hf_directory(str(tmp_path), kept=(kept,))
    out = str(tmp_path / "out.gguf")
    import_to_gguf(str(tmp_path), out, log=lambda s: None)
    model = Engine.load(out, "cpu", EngineOptions(max_ctx=256, max_seqs=1)).model
    x = torch.randn(5, 256, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    got = model.layers[0]["attn"].qkv(x).float()
    for lo, name in ((0, "q_proj"), (256, "k_proj")):
        w = dense[f"model.layers.0.self_attn.{name}"]
        want = x.float() @ w.t()
        have = got[:, lo:lo + w.shape[0]]
        # 2^-4 for codes of the rows, 2^-8 for the output and the file's 8-bit type of the kept matrix: another row order has nothing in common with it (error sqrt(2))
        assert float((have - want).norm() / want.norm()) < 0.1


def test_refusals_of_import(tmp_path):
    cfg = {"model_type": "llama", "hidden_size": 256, "num_hidden_layers": 1, "num_attention_heads": 4, "num_key_value_heads": 2, "intermediate_size": 384,
           "vocab_size": 320}
    for q in ({"quant_method": "fp8"}, {"quant_method": "fp8", "weight_block_size": [128, 64]}, {"quant_method": "fp8", "weight_block_size": [8, 128]},
              {"quant_method": "fp8", "weight_block_size": [128, 128], "activation_scheme": "static"}):
        with pytest.raises(ImportError_):
            parse_hf_config(json.dumps(dict(cfg, quantization_config=q)))
    assert parse_hf_config(json.dumps(dict(cfg, quantization_config={"quant_method": "fp8", "weight_block_size": [128, 128]}))).fp8_block == (128, 128)
    hf_directory(str(tmp_path), block=(256, 128))            # (scales of another block size than the file says)
    with pytest.raises(ImportError_):
        import_to_gguf(str(tmp_path), str(tmp_path / "x.gguf"), log=lambda s: None)


def prompt(cfg):
    return torch.randint(0, cfg.vocab, (150,), generator=torch.Generator().manual_seed(1)).tolist()


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["tiny-llama", "tiny-qwen3moe", "tiny-qwen3next"])
def test_generation_on_the_gpu_repeats_itself(name):
    """Prompts of several lengths together, then single tokens in captured graphs: every product's sums have a fixed order, so a second engine gives the same tokens."""
    cfg = preset(name)
    ids = prompt(cfg)
    runs = []
    for _ in range(2):
        eng = LLMEngine(build_model(cfg, torch.device("cuda:0"), quant="fp8", max_ctx=512), EngineOptions(max_ctx=512, max_batch_tokens=256, max_seqs=4, cuda_graphs=True))
        runs.append(eng.generate([ids, ids[:9], ids[:40]], SamplingParams(max_tokens=8)))
    assert runs[0] == runs[1] and all(len(o) == 8 for o in runs[0])


@pytest.mark.gpu
def test_logits_of_a_dense_model_against_the_cpu():
    """Both sides round activations to e4m3; where fp32 sums in another order end a bf16 step apart, a code may differ by one step of 2^-3 of its value.  Of the values
    that are a bf16 step (2^-8) off, about one in 2^-4 / 2^-8 = 16 lies that near to a border of e4m3, and fp32 sums that differ by 2^-22 cross a bf16 border once in
    2^14: a product's input is off by 2^-3 in less than 1e-4 of its elements, 2e-3 in norm after the square root, and four products a layer over a few layers, each
    passed on through norms, stay below 0.05, a cosine above 0.997."""
    from machx_inference_engine_b200.models.transformer import KV_BLOCK, ForwardBatch
    cfg = preset("tiny-llama")
    ids = prompt(cfg)
    res = {}
    for dev in ("cpu", "cuda:0"):
        d = torch.device(dev)
        m = build_model(cfg, d, quant="fp8", max_ctx=512, gen_device="cpu")
        kv = m.new_kv_cache(6)
        T = len(ids)
        pos = torch.arange(T, dtype=torch.int32, device=d)
        bt = torch.arange(1, 5, dtype=torch.int32, device=d).unsqueeze(0)
        slot = bt[0][(pos // KV_BLOCK).long()].long() * KV_BLOCK + (pos % KV_BLOCK).long()
        fb = ForwardBatch(torch.tensor(ids, dtype=torch.int32, device=d), pos, slot, bt, torch.tensor([T], dtype=torch.int32, device=d),
                          torch.tensor([0, T], dtype=torch.int32, device=d), T, logit_rows=torch.arange(T, device=d))
        res[dev] = m.forward(fb, kv).float().cpu()
    a, b = res["cpu"].flatten(), res["cuda:0"].flatten()
    assert float(torch.dot(a, b) / (a.norm() * b.norm())) > 0.997
