"""Models whose matrices are kept in 8 or 4 bits, through the step function and the Python entry point, against a plain forward pass in 64 bits
that is given the same quantised matrices (and quantises the rows of every product where the engine does)."""
import math

import pytest
import torch

import plain_llama
import replay_util as ru
from tiny_configs import CONFIGS, make_model_folder

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F64 = torch.float64


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    root = tmp_path_factory.mktemp("quant_models")
    return {n: make_model_folder(root, n) for n in CONFIGS}


def dense_weights(model):
    """What the engine's quantised matrices stand for, by checkpoint name (fp64, on the CPU)."""
    spec, out = model.spec, {}
    for i, (ls, b) in enumerate(zip(spec.layers, model.blocks)):
        p, m, f = f"model.layers.{i}.", b.mixer, b.feed_forward
        qkv = m.qkv.dense().double().cpu()
        n = [m.H * m.hs, m.KV * m.hs, m.KV * m.hs]
        for name, t in zip("qkv", qkv.split(n)):
            out[p + f"self_attn.{name}_proj.weight"] = t
        out[p + "self_attn.o_proj.weight"] = m.o.dense().double().cpu()
        gu = f.gate_up.dense().double().cpu().view(-1, 2, f.group, f.hidden)
        out[p + "mlp.gate_proj.weight"], out[p + "mlp.up_proj.weight"] = (gu[:, j].reshape(f.inter, f.hidden) for j in (0, 1))
        out[p + "mlp.down_proj.weight"] = f.down.dense().double().cpu()
    return out


def eight_bits(x):
    s = x.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -100) / 448
    return (x / s).float().to(torch.float8_e4m3fn).to(F64) * s


def plain_forward(cfg, w, tokens, q8, round_to=None):
    """``plain_llama.forward`` with the rows of a layer's products in 8 bits where ``q8`` says so."""
    H, KV = cfg["num_attention_heads"], cfg["num_key_value_heads"]
    hs, eps = cfg["head_dim"], cfg["rms_norm_eps"]
    rnd = (lambda t: t.to(round_to).to(F64)) if round_to is not None else (lambda t: t)
    rows = eight_bits if q8 else rnd                          # the 8-bit rows come straight from fp32
    pos = torch.arange(len(tokens))
    freqs = plain_llama.rope_frequencies(hs, cfg["rope_theta"], cfg.get("rope_scaling"))
    h = plain_llama.embedding(torch.as_tensor(list(tokens)), w["model.embed_tokens.weight"])
    for i in range(cfg["num_hidden_layers"]):
        p = f"model.layers.{i}."
        x = rows(plain_llama.rmsnorm(h, w[p + "input_layernorm.weight"], eps))
        q, k, v = (rnd(x @ w[p + f"self_attn.{n}_proj.weight"].T).view(-1, heads, hs) for n, heads in (("q", H), ("k", KV), ("v", KV)))
        q, k = rnd(plain_llama.rope(q, pos, freqs)), rnd(plain_llama.rope(k, pos, freqs))
        a = rnd(plain_llama.attention(q, k, v, 1.0 / math.sqrt(hs))).reshape(-1, H * hs)
        h = h + rnd((eight_bits(a) if q8 else a) @ w[p + "self_attn.o_proj.weight"].T)
        x = rows(plain_llama.rmsnorm(h, w[p + "post_attention_layernorm.weight"], eps))
        m = rows(plain_llama.swiglu(rnd(x @ w[p + "mlp.gate_proj.weight"].T), rnd(x @ w[p + "mlp.up_proj.weight"].T)))
        h = h + rnd(m @ w[p + "mlp.down_proj.weight"].T)
    x = rnd(plain_llama.rmsnorm(h, w["model.norm.weight"], eps))
    return x @ (w["model.embed_tokens.weight"] if cfg["tie_word_embeddings"] else w["lm_head.weight"]).T


@pytest.mark.parametrize("fmt", ["q8", "w4"])
@pytest.mark.parametrize("name", sorted(CONFIGS))
def test_logits_follow_the_plain_forward(folders, name, fmt):
    """Whole prompts, portions and single tokens. The error that rounding to bf16 makes is predicted by the plain pass itself (with bf16 roundings
    where the engine stores, against without); three times its largest is allowed, as for models without a format. In 8 bits a rounded row may
    also fall on the other side of a code's border; the prediction has those cases too, since its rows are rounded before they become codes."""
    from llm_steadyinfer_b200.engine.replay import Replayer
    cfg, _, page = CONFIGS[name]
    rp = Replayer(folders[name], torch.bfloat16, 512, page_size=page, weight_format=fmt)
    cfg, w = plain_llama.read_model_folder(folders[name])
    w.update(dense_weights(rp.runner.model))
    tokens = ru.random_tokens(cfg["vocab_size"], 150, 3)
    want = plain_forward(cfg, w, tokens, fmt == "q8")
    if fmt == "w4":                                             # and the rounding of a weight to bf16, which products of more than a few rows make
        rounded = {k: (t.to(torch.bfloat16).to(F64) if "_proj" in k else t) for k, t in w.items()}
    else:
        rounded = w
    allowed = 3 * (plain_forward(cfg, rounded, tokens, fmt == "q8", torch.bfloat16) - want).abs().max().item()
    worst = 0.0
    for cuts in ([150], [1, 7, 9, 16, 33, 84], [140] + [1] * 10):
        at = 0
        for n in cuts:
            got = rp.run_step([{"id": 0, "tokens": tokens[at:at + n], "want": list(range(n))}])
            worst = max(worst, (got.double() - want[at:at + n]).abs().max().item())
            at += n
        rp.run_step([], [0])
    assert worst <= allowed, f"{worst:.3e} (allowed {allowed:.3e})"


@pytest.mark.parametrize("fmt", ["q8", "w4"])
def test_generation_is_the_same_with_and_without_graphs(folders, fmt):
    """Greedy tokens of several requests: twice alike, and alike from recorded decode graphs and step by step."""
    from llm_steadyinfer_b200 import LLM, SamplingParams
    cfg = CONFIGS["C"][0]
    prompts = [ru.random_tokens(cfg["vocab_size"], n, 50 + n) for n in (3, 40, 77, 150)]
    out = []
    for graphs in (True, True, False):
        llm = LLM(folders["C"], dtype="bfloat16", max_batch=4, max_seq_len=256, max_gen_len=24, use_cuda_graph=graphs, async_decode=False, weight_format=fmt)
        out.append([r.token_ids for r in llm.generate(prompts, SamplingParams(ignore_eos=True))])
        assert all(len(t) == 24 for t in out[-1])
        assert llm.runner.graphs_available()
        if graphs:
            assert llm.stats["graph_steps"] > 0
    assert out[0] == out[1] == out[2]


def test_a_built_model_has_its_own_format(folders):
    from llm_steadyinfer_b200 import LLM
    from llm_steadyinfer_b200.weights import load_model
    model = load_model(folders["A"], torch.bfloat16, DEV, "w4")
    assert model.weight_format == "w4"
    LLM(model, dtype="bfloat16", max_batch=2, max_seq_len=64)
    with pytest.raises(ValueError, match="built model"):
        LLM(model, dtype="bfloat16", max_batch=2, max_seq_len=64, weight_format="w4")


def test_quantised_weights_stand_for_the_checkpoints(folders):
    """A matrix in 8 bits is off by half a step of e4m3 (2^-4 of an entry, 2^-10 of the row's scale near zero); in 4 bits by half a step of its group,
    and by what the zero point's rounding and the scale's (2^-8 of at most 15 steps) add."""
    from llm_steadyinfer_b200.parts.quantized import quantize
    g = torch.Generator(device=DEV).manual_seed(0)
    w = (torch.randn(96, 328, generator=g, device=DEV) * 0.02).to(torch.bfloat16)
    w[5] = 0
    w[6, 128:256] = 0.01                                         # a group on one side of zero
    q = quantize(w, "q8")
    off = (q.dense().double() - w.double()).abs()
    assert (off <= torch.maximum(w.double().abs() * 2.0 ** -4, q.scale.double().unsqueeze(1) * 2.0 ** -10) * (1 + 2.0 ** -20)).all()
    q = quantize(w, "w4")
    step = q.scales.double().repeat_interleave(128, 1)[:, :328]
    assert ((q.dense().double() - w.double()).abs() <= step * (0.5 + 0.5 + 15 * 2.0 ** -8)).all()
    assert (q.dense()[5] == 0).all()
