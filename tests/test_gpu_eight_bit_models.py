"""Parts and models with matrices in 8 bits.

A part's product of given activations is held to what roundings at borders allow: its input is quantised exactly as the plain form's; what lies
between two products is within 1e-5 of it (32-bit sums, the gate), so at most 1e-5 / 2^-4 * 2 of its entries are rounded to another neighbour, a
step of 2^-3 at most: 2-norm error sqrt(3.2e-4) * 2^-3 = 2.3e-3 of the result.  In a whole model such entries meet further roundings, until two
correct runs differ by the roundings themselves: 2^-4 / sqrt(3) of a value in the mean square, 0.036, and sqrt(2) of it between two runs, 0.051, for
every product of a branch; two products a branch, four branches, of which the stream is the sum: below 0.1 of the logits."""
import json
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from fp8_plain import gate_up_values, held, matrix_values, rows_values
from plain import qwen3_plain as P
from test_eight_bit_models import FP8, QWEN3, with_fp8
from test_gpu_kernels import DEV, rnd

pytestmark = pytest.mark.gpu
PART, MODEL = 2.3e-3, 0.1


def near(got, ref, most, what):
    err = float((got.double() - ref.double()).norm() / ref.double().norm())
    assert err <= most, f"{what}: {err:.2e} > {most}"


def make_part(kind, spec, hidden, seed, dtype):
    """A feed-forward of the library with random matrices, quantised, as a checkpoint's tensors are bound."""
    from gguf2bin_b200.config.specs import PartSpec
    from gguf2bin_b200.parts.registry import feed_forward_class
    from gguf2bin_b200.weights.random_init import random_tensors_on_device
    p = PartSpec.make(kind, eight_bit=True, **spec)
    cls = feed_forward_class(p)
    part = cls(p, hidden, dtype, DEV)
    part.bind(random_tensors_on_device(cls.expected(p, hidden), seed, torch.bfloat16, dtype, DEV, std=0.05))
    return part


def context(dtype):
    from gguf2bin_b200.engine.workspace import Workspace
    return SimpleNamespace(workspace=Workspace(DEV), dtype=dtype)


def feed_forward64(x, gu, down, q=None):
    """down(silu(gate x) * up x) of quantised rows, in 64 bits."""
    a = rows_values(*held(x))
    g, u = (a @ m.T for m in gate_up_values(gu.q, gu.scale))
    return rows_values(*held((g * torch.sigmoid(g) * u).float())) @ matrix_values(down.q, down.scale).T


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,inter,hidden", [(1, 264, 192), (16, 1024, 512), (17, 136, 130), (200, 640, 384), (700, 264, 192)])
def test_swiglu(T, inter, hidden, dtype):
    from gguf2bin_b200 import kernels_bf16
    part = make_part("swiglu", dict(intermediate_size=inter, names=(("gate", "g"), ("up", "u"), ("down", "d"))), hidden, 5, dtype)
    h = rnd(T, hidden, seed=T).to(dtype)
    ref = feed_forward64(h, part.w_gate_up, part.w_down)
    out = torch.full((T, hidden), 3.0, device=DEV)
    part.forward_into(h, context(dtype), out)
    near(out, ref, PART, "stored")
    base = rnd(T, hidden, seed=2)
    acc = base.clone()
    part.forward(h, context(dtype), acc)
    assert torch.equal(acc, base + out)
    kernels_bf16.check_status()
    assert part.notices() == [] and len(part.weights()) == 4


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,E,identity,top", [(1, 6, 0, 2), (9, 12, 3, 4), (150, 4, 1, 2), (600, 8, 0, 3)])
def test_routed_experts(T, E, identity, top, dtype):
    from gguf2bin_b200 import kernels, kernels_bf16
    hidden, inter = 320, 136
    names = (("router", "r"), ("gate", "e{}.g"), ("up", "e{}.u"), ("down", "e{}.d"))
    part = make_part("routed_experts", dict(n_experts=E, n_identity=identity, top=top, intermediate_size=inter, names=names), hidden, 6, dtype)
    h = rnd(T, hidden, seed=T).to(dtype)
    z = torch.empty(T, E + identity, device=DEV)
    kernels.linear(h, part.w_router, z)
    idx, weight = torch.empty(T, top, dtype=torch.int32, device=DEV), torch.empty(T, top, device=DEV)
    kernels.moe_route(z, None, top, False, idx, weight)
    ref = torch.zeros(T, hidden, dtype=torch.float64, device=DEV)
    for e in range(E + identity):
        token, choice = torch.nonzero(idx == e, as_tuple=True)
        if len(token):
            y = h[token].double() if e >= E else feed_forward64(
                h[token], SimpleNamespace(q=part.w_gate_up.q[e], scale=part.w_gate_up.scale[e]), SimpleNamespace(q=part.w_down.q[e], scale=part.w_down.scale[e]))
            ref.index_add_(0, token, y * weight[token, choice].double()[:, None])
    out = torch.full((T, hidden), 3.0, device=DEV)
    part.forward_into(h, context(dtype), out)
    near(out, ref, PART, "stored")
    base = rnd(T, hidden, seed=2)
    acc = base.clone()
    part.forward(h, context(dtype), acc)
    assert torch.equal(acc, base + out)
    kernels_bf16.check_status()


class Eight:
    """A matrix of the plain implementation: x @ W.T with x quantised."""
    __array_ufunc__ = None

    def __init__(self, q, scale):
        full = torch.zeros(q.shape[0], -(-q.shape[1] // 128) * 128, dtype=torch.uint8)
        full[:, :q.shape[1]] = torch.from_numpy(q)
        self.w = matrix_values(full.view(torch.float8_e4m3fn), torch.from_numpy(scale)).numpy()
        self.T = self

    def astype(self, dt):
        return self

    def __rmatmul__(self, x):
        return (rows_values(*held(torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)))).numpy() @ self.w.T).astype(x.dtype)


def plain(folder):
    from gguf2bin_b200.weights.safetensors_io import SafetensorsFile
    f = SafetensorsFile(folder / "model.safetensors")
    W = {}
    for n, e in f.entries.items():
        if n.endswith("_scale_inv"):
            continue
        t = f.tensor(n)
        W[n] = Eight(t.view(torch.uint8).numpy(), f.tensor(n + "_scale_inv").float().numpy()) if e.dtype == "F8_E4M3" else t.float().numpy()
    cfg = json.loads((folder / "config.json").read_text())
    return lambda tokens: P.forward(cfg, W, list(tokens), np.float32)


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    from gguf2bin_b200.weights import write_random_model
    return write_random_model(tmp_path_factory.mktemp("eight") / "m", with_fp8(), 4)


# heads of 64: k and v end inside blocks of 128 in the second configuration (three products side by side)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("kv", [2, 1])
def test_a_model_beside_the_plain_implementation(dtype, kv, tmp_path):
    from gguf2bin_b200.api import LLM, StepEntry
    from gguf2bin_b200.weights import write_random_model
    where = write_random_model(tmp_path / "m", dict(with_fp8(), num_key_value_heads=kv, num_attention_heads=3 if kv == 1 else 4), 4, std=0.05)
    tokens = np.random.default_rng(1).integers(0, 311, 150).tolist()
    ref = torch.from_numpy(plain(where)(tokens))
    llm = LLM(where, dtype=dtype, max_tokens=512)
    seq = llm.open_sequence()
    whole = llm.step([StepEntry(seq, tokens, range(150))]).cpu()
    near(whole, ref, MODEL, "one prompt")
    other = llm.open_sequence()
    rows = [llm.step([StepEntry(other, tokens[:130], range(130))]).cpu()]
    for i in range(130, 150):
        rows.append(llm.step([StepEntry(other, tokens[i:i + 1], [0])]).cpu())
    near(torch.cat(rows), ref, MODEL, "a prompt, then token after token")


def test_generation_and_random_models(folder):
    """A model made on the device is the one that the folder holds, batches generate (graphs, rows of padding), and generation repeats itself."""
    from gguf2bin_b200.api import LLM, StepEntry
    prompts = [np.random.default_rng(i).integers(0, 311, n).tolist() for i, n in enumerate((40, 3, 17, 1, 9, 64, 25, 2, 30))]
    how = dict(n=12, temperature=0.0, top_k=0, top_p=1.0, repeat_penalty=1.0, ignore_eos=True)
    made = LLM.random(with_fp8(), seed=4, max_tokens=2048)
    loaded = LLM(folder, dtype="bfloat16", max_tokens=2048)
    outs = [[o.tokens for o in m.generate(prompts, **how)] for m in (made, loaded, loaded)]
    assert outs[0] == outs[1] == outs[2] and all(len(t) == 12 for t in outs[0])
    forward = plain(folder)
    seq = loaded.open_sequence()
    full = prompts[0] + outs[0][0]
    logits = loaded.step([StepEntry(seq, full, range(len(full)))]).cpu()
    ref = torch.from_numpy(forward(full))
    near(logits, ref, MODEL, "what was generated")
    held_bytes, plain_bytes = loaded.model.weight_bytes(), LLM.random(QWEN3, seed=4, max_tokens=64).model.weight_bytes()
    assert held_bytes < 0.8 * plain_bytes


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_routed_architecture(dtype):
    """Levolix with its experts and its chunked attention's matrices in 8 bits generates and repeats itself."""
    import levolix_helpers as L
    from gguf2bin_b200.api import LLM
    cfg = dict(L.CONFIGS["u"], quantization_config=FP8)
    llm = LLM.random(cfg, seed=2, max_tokens=1024, dtype=dtype)
    how = dict(n=8, temperature=0.0, top_k=0, top_p=1.0, repeat_penalty=1.0, ignore_eos=True)
    prompts = [[3, 5, 7, 1, 2], [9] * 40]
    first = [o.tokens for o in llm.generate(prompts, **how)]
    assert first == [o.tokens for o in llm.generate(prompts, **how)] and all(len(t) == 8 for t in first)
    assert any(getattr(b.feed_forward, "eight_bit", False) for b in llm.model.blocks)
