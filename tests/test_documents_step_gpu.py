"""The document attention and the token embedding as the decoder uses them: whole updates with
`Runtime.attention = "documents"` and a trained embedding, against the reference's fixtures and the oracle."""

import numpy as np
import pytest
import torch

from causal_tuner_b200.modeling.config import ModelConfig
from causal_tuner_b200.modeling.model import CausalLM, Runtime
from causal_tuner_b200.training import Trainer, make_optimizer
from oracle import model as oracle_model
from test_step_gpu import CONFIG, batch_of, load_model

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("gpu_guard")]

FP32 = dict(base_dtype=torch.float32, train_dtype=torch.float32, compute_dtype=torch.float32)


@pytest.mark.parametrize("checkpoint", [False, True])
def test_fp32_step_matches_the_reference_fixture(golden, checkpoint):
    g = golden("step_tiny_b1.npz")
    model = load_model(g, Runtime(rank=16, attention="documents", checkpoint=checkpoint, **FP32), nf4=False)
    metrics = Trainer(model, make_optimizer(model, learning_rate=1e-4), device="cuda", loss_token_budget=128).update([batch_of(g)])
    # the bounds of the same step with "vanilla" attention (test_step_gpu.py)
    assert abs(metrics["loss"] - float(g["loss"])) / float(g["loss"]) < 1e-5
    assert abs(metrics["grad_norm"] - float(g["grad_norm"])) / float(g["grad_norm"]) < 1e-3
    for name, parameter in model.named_parameters():
        if parameter.requires_grad:
            expected = torch.from_numpy(g["g__" + name.replace(".", "__")])
            scale = expected.abs().max().item()
            torch.testing.assert_close(parameter.grad.cpu(), expected, rtol=2e-3, atol=2e-4 * scale + 1e-9, msg=name)


def test_bf16_nf4_step_tracks_the_bf16_reference_fixture(golden):
    g = golden("step_tiny_bf16.npz")
    runtime = Runtime(rank=16, base_dtype=torch.float32, compute_dtype=torch.bfloat16, attention="documents", checkpoint=True)
    model = load_model(g, runtime, nf4=True)
    metrics = Trainer(model, make_optimizer(model, learning_rate=1e-4), device="cuda").update([batch_of(g)])
    # the bounds of the same step with the library's attention (test_step_gpu.py)
    assert abs(metrics["loss"] - float(g["loss"])) / float(g["loss"]) < 1e-3
    assert abs(metrics["grad_norm"] - float(g["grad_norm"])) / float(g["grad_norm"]) < 2e-2
    trained = [(n, p) for n, p in model.named_parameters() if p.requires_grad]
    actual = torch.cat([p.grad.flatten().cpu() for _, p in trained])
    expected = torch.cat([torch.from_numpy(g["g__" + n.replace(".", "__")]).flatten() for n, _ in trained])
    assert ((actual - expected).norm() / expected.norm()).item() < 5e-2


def padded_batch(g):
    """The fixture's batch with padding inside and behind the documents."""
    batch = batch_of(g)
    batch["attention_mask"][0, 100:117] = 0
    batch["attention_mask"][0, 480:] = 0
    batch["attention_mask"][1, :3] = 0
    return batch


def gradients(model, batch):
    from causal_tuner_b200.kernels.loss import active_rows, projection_loss
    from causal_tuner_b200.segments import prediction_targets
    targets, weights = prediction_targets(batch)
    rows = active_rows(weights, "cuda")
    hidden = model({k: v.cuda() for k, v in batch.items()})
    loss = projection_loss(hidden, model.lm_head.weight, targets.cuda(), weights.cuda(), token_budget=128,
                           compute_dtype=model.runtime.compute_dtype, rows=rows)
    parameters = [(n, p) for n, p in model.named_parameters() if p.requires_grad]
    grads = torch.autograd.grad(loss, [p for _, p in parameters])
    return float(loss.detach()), {n: grad for (n, _), grad in zip(parameters, grads)}


@pytest.mark.parametrize("scale", [1.0, 16.0])
def test_a_trained_embedding_and_padding_against_the_oracle(golden, scale):
    g = golden("step_tiny_b1.npz")
    batch = padded_batch(g)
    runtime = Runtime(rank=16, attention="documents", train_embed=True, **FP32)
    model = load_model(g, runtime, nf4=False)
    model.config = ModelConfig(**CONFIG, embed_scale=scale)
    loss, grads = gradients(model, batch)
    table = model.model.embed_tokens.weight
    assert table.requires_grad and grads["model.embed_tokens.weight"].dtype == torch.float32
    params = {n: p.detach().cpu().clone() for n, p in model.named_parameters()}
    leaf = params["model.embed_tokens.weight"].requires_grad_(True)
    expected_loss, _ = oracle_model.step_loss(
        {**params, "model.embed_tokens.weight": leaf * scale}, batch, layers=2, heads=4, head_dim=64, rotary_dim=32, theta=1e4, eps=1e-5)
    expected, = torch.autograd.grad(expected_loss, leaf)
    expected[CONFIG["pad_token_id"]] = 0                     # the module's padding row gets no gradient
    assert abs(loss - float(expected_loss)) / abs(float(expected_loss)) < 1e-5
    actual = grads["model.embed_tokens.weight"].cpu()
    peak = expected.abs().max().item()
    torch.testing.assert_close(actual, expected, rtol=2e-3, atol=2e-4 * peak)
    seen = torch.zeros(CONFIG["vocab_size"], dtype=torch.bool)
    seen[batch["input_ids"].flatten()] = True
    assert (actual[~seen] == 0).all()


def test_documents_agree_with_the_other_attention_settings(golden):
    """fp32: the dense form; bf16: the library's kernels, by way of gather and scatter for the padding."""
    g = golden("step_tiny_b1.npz")
    batch = padded_batch(g)
    for other, dtypes, loss_bound, grad_bound in (("vanilla", FP32, 1e-5, 1e-4),
                                                  ("flash_attention_2", dict(base_dtype=torch.bfloat16), 1e-3, 5e-2)):
        if other == "flash_attention_2":
            pytest.importorskip("flash_attn")
        results = []
        for attention in ("documents", other):
            model = load_model(g, Runtime(rank=16, attention=attention, **dtypes), nf4=False)
            results.append(gradients(model, batch))
        (loss, grads), (other_loss, other_grads) = results
        assert abs(loss - other_loss) <= loss_bound * abs(other_loss)
        a = torch.cat([grads[n].flatten() for n in grads]).double()
        b = torch.cat([other_grads[n].flatten() for n in grads]).double()
        assert float((a - b).norm() / b.norm()) < grad_bound


def test_updates_are_reproducible(golden):
    g = golden("step_tiny_b1.npz")

    def run():
        model = load_model(g, Runtime(rank=16, base_dtype=torch.bfloat16, attention="documents", train_embed=True), nf4=True)
        trainer = Trainer(model, make_optimizer(model, learning_rate=1e-3), device="cuda")
        losses = [trainer.update([padded_batch(g), batch_of(g)])["loss"] for _ in range(3)]
        return losses, [p.detach().clone() for p in model.parameters() if p.requires_grad]
    (first, values), (second, again) = run(), run()
    assert first == second and all(torch.equal(a, b) for a, b in zip(values, again))
    assert np.isfinite(first).all()


def test_hooks_on_the_embedding_run(golden):
    g = golden("step_tiny_b1.npz")
    batch = {k: v.cuda() for k, v in batch_of(g).items()}
    model = load_model(g, Runtime(rank=16, attention="documents", **FP32), nf4=False)
    with torch.no_grad():
        expected = model(batch)
        seen = []
        handle = model.model.embed_tokens.register_forward_hook(lambda module, args, out: seen.append(out.clone()) or 2 * out)
        changed = model(batch)
        handle.remove()
        assert torch.equal(model(batch), expected) and not torch.equal(changed, expected)
        table = model.model.embed_tokens
        assert len(seen) == 1 and torch.equal(seen[0], table.weight[batch["input_ids"]])
        assert torch.equal(table(batch["input_ids"]), seen[0])          # the module on its own


def test_an_attention_block_without_a_prepared_layout(golden):
    """As the library's form does, the block makes the plan from the spans it is given."""
    from causal_tuner_b200.kernels.attention_cuda import prepare_documents
    from causal_tuner_b200.modeling.rotary import rotary_values
    from causal_tuner_b200.segments import canonical_segments, position_ids, runs
    g = golden("step_tiny_b1.npz")
    batch = {k: v.cuda() for k, v in batch_of(g).items()}
    model = load_model(g, Runtime(rank=16, attention="documents", **FP32), nf4=False)
    segments = canonical_segments(batch["attention_mask"], batch.get("segment_ids"))
    spans, c = runs(segments), model.config
    rotary = rotary_values(position_ids(segments), c, torch.float32)
    with torch.no_grad():
        x = model.model.embed_tokens(batch["input_ids"], 1.0, torch.float32)
        block = model.model.layers[0].self_attn
        plan = prepare_documents(x.shape[:2], spans, x.device, c.num_attention_heads, c.num_key_value_heads)
        residual = torch.zeros_like(x)
        results = [block(x, *rotary, segments, spans, layout, residual=residual) for layout in (None, plan)]
    assert torch.equal(*results)
