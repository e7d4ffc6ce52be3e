"""Scoring of texts: windows, contexts and the command against log probabilities worked out token by token."""
import json
import math

import pytest
import torch

from tnn_b200 import cli
from tnn_b200.inference import score_tokens
from tnn_b200.models import zoo


def _by_hand(g, ids, S, context, temperature):
    """(log probability, entropy, logits) of ids[1:], each from the window that predicts it."""
    out, at, done = [], 0, 1
    while done < len(ids):
        window = ids[at:at + S]
        x = torch.zeros(1, S, dtype=torch.long)
        x[0, :len(window)] = torch.tensor(window)
        logits = g.forward({"input": x.to(g.device)})["output"][0].double().cpu()
        for pos in range(len(window)):
            if at + pos + 1 == done and done < len(ids):
                lp = torch.log_softmax(logits[pos] / temperature, 0)
                out.append((float(lp[ids[done]]), float(-(lp.exp() * lp).sum()), logits[pos]))
                done += 1
        at += S - context
    return out


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("n,context", [(2, None), (16, None), (17, None), (18, 0), (40, None), (50, 15), (33, 3)])
def test_windows(dev, n, context):
    S = 16 if dev == "cpu" else 64
    n = n if dev == "cpu" else 4 * n
    g = zoo.gpt2(64, 1, 2, "t", seq_len=S, vocab=97, drop=0.0).compile(device=dev, seed=2)
    ids = torch.randint(0, 97, (n,), generator=torch.Generator().manual_seed(n)).tolist()
    r = score_tokens(g, ids, 4, 0.8, context=context, batch=3)
    g.set_training(False)
    ref = _by_hand(g, ids, S, S // 2 if context is None else context, 0.8)
    assert r.log_probs.shape == (n - 1,) and r.top_indices.shape == (n - 1, 4)
    for i, (lp, ent, logits) in enumerate(ref):
        assert abs(float(r.log_probs[i]) - lp) < 1e-4 and abs(float(r.entropy[i]) - ent) < 1e-4
        assert torch.equal(r.top_indices[i].cpu(), torch.sort(logits.float(), descending=True, stable=True).indices[:4])


def test_refusals():
    g = zoo.gpt2(64, 1, 1, "t", seq_len=8, vocab=20).compile(device="cpu", seed=0)
    for args in (dict(tokens=[3]), dict(tokens=[3, 4], context=8), dict(tokens=[3, 4], batch=0), dict(tokens=[3, 4], top_k=21)):
        with pytest.raises(ValueError):
            score_tokens(g, **args)


def test_training_mode_is_put_back():
    g = zoo.gpt2(64, 1, 1, "t", seq_len=8, vocab=20).compile(device="cpu", seed=0)
    g.set_training(True)
    score_tokens(g, [1, 2, 3])
    assert g.training


def test_command(capsys, tmp_path):
    path = str(tmp_path / "m.tnng")
    zoo.gpt2(64, 1, 1, "t", seq_len=8, vocab=20).compile(device="cpu", seed=0).save_state(path)
    assert cli.main(["score", "--model-path", path, "--token-ids", "1,2,3,4,5,6,7,8,9,10,11", "--top", "2", "--device", "CPU"]) == 0
    lines = capsys.readouterr().out.strip().splitlines()
    summary = json.loads(lines[-1])
    assert len(lines) == 11 and summary["tokens"] == 10
    assert abs(summary["perplexity"] - math.exp(-summary["mean_log_prob"])) < 1e-6 * summary["perplexity"]


def test_tokens_outside_the_vocabulary_are_refused():
    g = zoo.gpt2(64, 1, 1, "t", seq_len=8, vocab=20).compile(device="cpu", seed=0)
    for tokens in ([3, -1, 2], [3, -100, 2], [20, 1], [1, 2, 20]):
        with pytest.raises(ValueError):
            score_tokens(g, tokens)
