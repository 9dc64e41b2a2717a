"""The output-head operators at work: perplexity without logits, the dense
model's top logits, tuning of a quantized model's final norm and head."""
import pytest
import torch

pytest.importorskip("transformers")
pytestmark = pytest.mark.gpu


def _model(kind, **kw):
    from test_gpu_stack import tiny_model
    return tiny_model(kind, **kw)


@pytest.mark.parametrize("kind", ["opt", "llama"])
def test_fused_perplexity(kind):
    """Against 64-bit losses of the same hidden states: only fp32 rounding of
    logits (200 tokens, 128 channels) and sums; and against the default, which
    rounds logits and losses to 16 bits."""
    from crb_amd.evaluate import eval_ppl, final_hidden, split_head
    m = _model(kind)
    ids = torch.randint(0, 200, (1, 5 * 64 + 9), generator=torch.Generator().manual_seed(3)).cuda()
    ppl, nll = eval_ppl(m, ids, 64, chunk=2, fused=True, return_nlls=True)
    w = ids[:, :5 * 64].reshape(5, 64)
    with torch.no_grad():
        h = final_hidden(m, w, 2)
        mods, head, scale = split_head(m)
        for x in mods:
            h = x(h)
        logq = torch.log_softmax(h.double() @ head.weight.double().t() / scale, -1)
    want = -logq[:, :-1].gather(2, w[:, 1:, None])[..., 0].mean(1) * 64
    assert float(((nll.double() - want) / want).abs().max()) < 1e-5
    assert ppl == pytest.approx(float((want.sum() / (5 * 64)).exp()), rel=1e-4)
    # a loss near 5.3 in bf16 is within 2^-8 of it
    assert eval_ppl(m, ids, 64, chunk=2) == pytest.approx(ppl, rel=3e-2)


@pytest.mark.parametrize("kind", ["opt", "llama"])
def test_teacher_top_is_the_models(kind):
    from crb_amd.recover import teacher_top
    m = _model(kind)
    w = torch.randint(0, 200, (3, 40), generator=torch.Generator().manual_seed(4)).cuda()
    top = teacher_top(m, w, k=9, chunk=3)
    with torch.no_grad():
        logits = m(w).logits
    assert top.val.shape == (3, 40, 9) and top.lse.shape == (3, 40)
    # the same model in other batches: within a few roundings of the logits' type
    u = 2.0 ** (-8 if logits.dtype == torch.bfloat16 else -11)
    z = logits.float().gather(2, top.idx.long())
    assert float((z - top.val.float()).abs().max()) <= 8 * u * float(logits.abs().max())
    lse = torch.logsumexp(logits.float(), -1)
    assert float((lse - top.lse).abs().max()) <= 8 * u * float(logits.abs().max()) + 1e-5


@pytest.mark.parametrize("kind,pack", [("opt", False), ("opt", True), ("llama", False)])
def test_recover_lowers_the_divergence(kind, pack):
    from crb_amd.evaluate import eval_ppl
    from crb_amd.recover import recover_head, teacher_top
    from crb_amd.stack import StackQuantizer
    from test_gpu_stack import _samples
    m = _model(kind)
    w = _samples(n=6, seq=96)
    top = teacher_top(m, w, k=32)
    StackQuantizer(m, chunk=3, pack=pack).run(w)
    layers = [p.detach().clone() for n, p in m.named_parameters() if ".layers." in n]
    losses = recover_head(m, w, top, steps=25, lr=1e-3, batch=6)
    assert all(x == x and x >= -1e-4 for x in losses)
    assert losses[-1] < 0.8 * losses[0], (losses[0], losses[-1])
    after = [p for n, p in m.named_parameters() if ".layers." in n]
    assert all(torch.equal(a, b) for a, b in zip(layers, after))
    emb = m.get_input_embeddings().weight
    assert emb is not m.get_output_embeddings().weight
    assert 1.0 < eval_ppl(m, w.reshape(1, -1), 96, fused=True) < 1e4


def test_command_line_with_recovery(capsys):
    from crb_amd import run
    out = run.main(["tiny-opt", "synthetic", "crb", "--nsamples", "4", "--seqlen", "64",
                    "--salient_metric", "hessian", "--recover_steps", "6", "--recover_topk", "16",
                    "--recover_lr", "1e-3", "--eval_tokens", "200", "--fused_eval"])
    assert len(out["recover_losses"]) == 6
    assert out["recover_losses"][-1] < out["recover_losses"][0]
    assert 1.0 < out["ppl"] < 1e4
    assert "recovery: KL" in capsys.readouterr().out
