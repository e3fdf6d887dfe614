"""The ribosomal autoencoder's uses of the token operators: scores of decoded positions (model, codec) and learning from
another autoencoder's best tokens (loss, trainer, command line)."""
import copy
import json
import os

import numpy as np
import pytest
import torch

from serann.genome.codec import RiboAECodec
from serann.genome.tokenizer import Vocabulary
from serann.models.riboae import ConcreteGAE, build_model
from serann.riboae import trainer as T
from serann.riboae.io import save_checkpoint

from . import token_oracle as O


def _model(seed=0, kind="concrete", V=12):
    torch.manual_seed(seed)
    m = build_model(kind, genotype_length=20, max_phenotype_length=32, vocabulary_size=V, embedding_dim=16)
    with torch.no_grad():
        for b in m.modules():
            if isinstance(b, torch.nn.BatchNorm1d):
                b.running_mean.normal_(0, 0.1)
                b.running_var.uniform_(0.5, 1.5)
    return m.eval()


def _bits(n, seed=3):
    return np.random.default_rng(seed).integers(0, 2, (n, 20))


def test_score_tokens_rates_every_position():
    m = _model()
    bits = _bits(5)
    r = m.score_tokens(bits, top_k=4, temperature=1.5)
    np.testing.assert_array_equal(r["tokens"], m.decode_tokens(bits))
    with torch.no_grad():
        z = torch.nn.functional.one_hot(torch.as_tensor(bits), 2).float()
        x = m.generative_net.logits(z).reshape(-1, 12)
    ref = O.score(x, torch.as_tensor(r["tokens"]).reshape(-1), 1.5, 4, -100)
    assert r["logprob"].shape == r["entropy"].shape == (5, 32) and r["top_ids"].shape == (5, 32, 4)
    np.testing.assert_array_equal(r["top_ids"].reshape(-1, 4), ref["top_ids"].numpy())
    tol = 64 * O.U * 20
    np.testing.assert_allclose(r["logprob"].reshape(-1), ref["logprob"].numpy(), rtol=tol, atol=tol)
    np.testing.assert_allclose(r["entropy"].reshape(-1), ref["entropy"].numpy(), rtol=tol, atol=tol)
    np.testing.assert_array_equal(r["top_ids"][..., 0], r["tokens"])
    given = np.zeros((5, 32), np.int64)
    assert "top_ids" not in m.score_tokens(bits, given)
    np.testing.assert_array_equal(m.score_tokens(bits, given)["tokens"], given)


def test_codec_scores_in_batches():
    m = _model()
    vocab = Vocabulary.build([[f"t{i}" for i in range(11)]])
    c = RiboAECodec(m, vocab, max_tokens=32, batch_size=4)
    bits = _bits(11)
    r = c.score_sequences(bits, top_k=3)
    np.testing.assert_array_equal(r["tokens"], c.decode_to_sequence(bits))
    want = m.score_tokens(bits, top_k=3)
    for k in want:
        np.testing.assert_array_equal(r[k], want[k])
    assert c.score_sequences(bits[0])["logprob"].shape == (1, 32)
    assert c.score_sequences(bits[:0], top_k=2)["top_ids"].shape == (0, 32, 2)


@pytest.mark.parametrize("kind", ["concrete", "deterministic"])
def test_loss_against_a_teacher(kind):
    """The reconstruction term becomes the divergence from the teacher's tokens; the gradient is the formula's."""
    teacher, m = _model(1), _model(2, kind).train()
    x = torch.randint(0, 12, (6, 32), generator=torch.Generator().manual_seed(5))
    u = torch.rand(6, 20, 2, generator=torch.Generator().manual_seed(6))
    taught = teacher.distill_targets(x, 5, 2.0)
    assert taught[0].shape == taught[1].shape == (6, 32, 5) and taught[2] == 2.0
    kw = dict(noise=u) if kind == "concrete" else {}
    plain = m.compute_loss(x, 0.3, 0.05, **kw)
    out = m.compute_loss(x, 0.3, 0.05, teacher=taught, **kw)
    assert torch.equal(out["nll"], plain["nll"]) and torch.equal(out["kld"], plain["kld"])
    z = m._encode(x, 0.3, u)[0] if kind == "concrete" else m._encode(x)
    logits = m.generative_net.logits(z).reshape(-1, 12)
    div, dx = O.distill(logits.detach(), taught[0].reshape(-1, 5), taught[1].reshape(-1, 5), 2.0, "drop", None)
    want = float(div.sum().detach()) / 6 + 0.05 * float(out["kld"].detach())
    # fp32 sums of 32 positions and 6 rows, and the division: 40 roundings of the terms' size
    assert abs(float(out["loss"].detach()) - want) <= 40 * O.U * (float(div.abs().sum()) / 6 + abs(0.05 * float(out["kld"].detach())))
    got, = torch.autograd.grad(out["loss"], m.generative_net.bn2.bias)
    total = dx.sum(0) / 6
    assert torch.allclose(got.double(), total, rtol=0, atol=200 * O.U * float(dx.abs().sum()) / 6)


@pytest.mark.parametrize("kind", ["concrete", "deterministic"])
def test_a_teacher_leaves_the_moving_statistics_of_a_step(kind):
    """The decoder runs once a step, with and without a teacher: its BatchNorm layers take the batch's statistics in once."""
    x = torch.randint(0, 12, (6, 32), generator=torch.Generator().manual_seed(5))
    kw = dict(noise=torch.rand(6, 20, 2, generator=torch.Generator().manual_seed(6))) if kind == "concrete" else {}
    taught = _model(1).distill_targets(x, 5, 2.0)
    plain, learner = _model(2, kind).train(), _model(2, kind).train()
    plain.compute_loss(x, 0.3, 0.05, **kw)
    learner.compute_loss(x, 0.3, 0.05, teacher=taught, **kw)
    for (name, a), (_, b) in zip(plain.named_buffers(), learner.named_buffers()):
        assert torch.equal(a, b), name


def test_scores_and_targets_leave_a_model_in_its_mode():
    """Asked in the middle of training, a model goes on with batch statistics; its answers are those of eval mode."""
    m = _model(1)
    x, bits = torch.randint(0, 12, (6, 32), generator=torch.Generator().manual_seed(5)), _bits(4)
    want, scored = m.distill_targets(x, 3), m.score_tokens(bits, top_k=2)
    m.train()
    m.generative_net.bn1.eval()
    got, again = m.distill_targets(x, 3), m.score_tokens(bits, top_k=2)
    assert m.training and m.generative_net.bn2.training and not m.generative_net.bn1.training
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for k in scored:
        np.testing.assert_array_equal(again[k], scored[k])
    with pytest.raises(ValueError):
        m.score_tokens(bits, top_k=13)
    assert m.training


def test_trainer_learns_from_a_teacher(tmp_path):
    teacher, m = _model(1), _model(2)
    before = copy.deepcopy(teacher.state_dict())
    data = np.random.default_rng(0).integers(0, 12, (48, 32))
    hist = T.train("kd", m, data, None, str(tmp_path), batch_size=16, max_steps=4, log=lambda *a: None, teacher=teacher,
                   teacher_top_k=3, distill_temperature=2.0)
    assert len(hist) == 4 and np.isfinite(hist).all()
    assert all(torch.equal(a, b) for a, b in zip(before.values(), teacher.state_dict().values()))
    for kw in (dict(teacher=_model(1, V=13)), dict(teacher=m), dict(teacher=teacher, teacher_top_k=0),
               dict(teacher=teacher, teacher_top_k=13)):
        with pytest.raises(ValueError):
            T.train("kd", m, data, None, str(tmp_path), batch_size=16, max_steps=1, log=lambda *a: None, **kw)


def test_training_command_with_a_teacher(tmp_path, monkeypatch):
    from serann.cli import tools
    monkeypatch.setitem(tools.riboae_config, "ribosomal_autoencoders_dir", str(tmp_path))
    save_checkpoint(tmp_path / "t.pt", _model(1), "concrete", 1)
    vocab = Vocabulary.build([[f"t{i}" for i in range(11)]])
    assert len(vocab) == 12
    vocab.save_csv(tmp_path / "v.csv")
    np.savez(tmp_path / "d.npz", sequences=np.random.default_rng(0).integers(0, 12, (20, 32)))
    params = {"batch_size": 8, "embedding_size": 16, "genotype_alphabet_size": 2, "genotype_size": 20,
              "min_backup_interval": 1000, "prior_temperature": 0.1, "source_code_length": 32, "train_test_ratio": 0.9}
    (tmp_path / "p.json").write_text(json.dumps(params))
    tools.training_main(["-p", str(tmp_path / "p.json"), "-n", "s", "--dataset", str(tmp_path / "d.npz"), "--vocabulary",
                         str(tmp_path / "v.csv"), "--max-steps", "2", "--device", "cpu", "--teacher", str(tmp_path / "t.pt"),
                         "--teacher-top-k", "4", "--distill-temperature", "1.5"])
    assert os.path.exists(tmp_path / "s_b2.pt")


# ------------------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_gpu_scores_follow_the_decoder():
    """On a GPU the positions are scored from the HIP decoder's logits.  A log-softmax moves by at most twice the largest
    change of its logits, so the scores agree with the CPU's within twice the logits' difference (and the fp32 bound)."""
    m = _model()
    bits = _bits(70)
    want = m.score_tokens(bits, top_k=3)
    with torch.no_grad():
        x = m.generative_net.logits(torch.nn.functional.one_hot(torch.as_tensor(bits), 2).float())
    g = copy.deepcopy(m).cuda()
    got = g.score_tokens(bits, want["tokens"], device="cuda", top_k=3)
    xg = g._eval_logits(torch.as_tensor(bits).cuda()).cpu()
    off = float((xg - x).abs().max())
    assert off < 0.1 * float(x.abs().max())
    assert np.abs(got["logprob"] - want["logprob"]).max() <= 2 * off + 1e-4
    ref = O.score(xg.reshape(-1, 12), torch.as_tensor(want["tokens"]).reshape(-1), 1.0, 3, -100)
    np.testing.assert_array_equal(got["top_ids"].reshape(-1, 3), ref["top_ids"].numpy())
    tol = O.sum_error(xg.reshape(-1, 12), 1.0) + 6 * O.U * 40
    np.testing.assert_allclose(got["logprob"].reshape(-1), ref["logprob"].numpy(), rtol=0, atol=tol)


@pytest.mark.gpu
def test_gpu_teacher_targets_match_the_cpu_where_the_codes_agree():
    m = _model(1)
    x = torch.randint(0, 12, (40, 32), generator=torch.Generator().manual_seed(2))
    g = copy.deepcopy(m).cuda()
    ids, lp, t = g.distill_targets(x.cuda(), 4, 1.5)
    bits_c, bits_g = m.encode(x), g._hip_encoder(x.cuda()).cpu()
    xg = g._eval_logits(bits_g.cuda()).reshape(-1, 12).cpu()
    ref = O.score(xg, None, 1.5, 4, -100)
    assert torch.equal(ids.reshape(-1, 4).cpu(), ref["top_ids"]) and t == 1.5
    assert float((bits_c == bits_g).float().mean()) > 0.9


@pytest.mark.gpu
def test_hip_step_against_a_teacher_matches_the_fp32_oracle(monkeypatch):
    """Every parameter gradient of a HIP step that learns from a teacher against the fp32 CPU model, with the bounds of the
    step that learns from tokens (5 %, cosine > 0.998, an absolute floor of 0.2 % of the largest element)."""
    from serann.riboae.hip_trainer import HipRiboTrainer

    from .test_riboae_hip_train import SPEC_OF, _err
    torch.manual_seed(0)
    m = ConcreteGAE(genotype_length=20, max_phenotype_length=32, vocabulary_size=12, embedding_dim=16, prior_temperature=0.1)
    g = torch.Generator().manual_seed(1)
    x, u = torch.randint(0, 12, (48, 32), generator=g), torch.rand(48, 20, 2, generator=g)
    taught = _model(1).distill_targets(x, 5, 2.0)
    monkeypatch.setenv("SERANN_RIBOAE_HIP", "0")
    c = copy.deepcopy(m).train()
    out = c.compute_loss(x, 0.3, 0.05, noise=u, teacher=taught)
    gr = torch.autograd.grad(out["loss"], list(c.parameters()))
    ref = {n: t.numpy().astype(np.float64) for (n, _), t in zip(c.named_parameters(), gr)}
    monkeypatch.delenv("SERANN_RIBOAE_HIP")
    tr = HipRiboTrainer(m.cuda().train(), device="cuda")
    dev = (taught[0].cuda(), taught[1].cuda(), taught[2])
    hip, res = tr.debug_grads(x.cuda(), 0.3, 0.05, u.cuda(), teacher=dev)
    again, res2 = tr.debug_grads(x.cuda(), 0.3, 0.05, u.cuda(), teacher=dev)
    assert res == res2 and all(np.array_equal(hip[k], again[k]) for k in hip)
    loss, kld = float(out["loss"].detach()), float(out["kld"].detach())
    assert abs(res["loss"] - loss) < 1e-2 * abs(loss) and abs(res["kld"] - kld) < 1e-2 * abs(kld) + 1e-3
    gmax = max(float(np.abs(v).max()) for v in ref.values())
    for k, tname in SPEC_OF.items():
        want, got = ref[tname], hip[k]
        if np.linalg.norm(want) < 1e-4 * gmax * np.sqrt(want.size):
            assert np.abs(got).max() < 1e-2 * gmax, k
            continue
        if np.linalg.norm(got - want) < 2e-3 * gmax * np.sqrt(want.size):
            continue
        e, cos = _err(got, want)
        assert e < 0.05 and cos > 0.998, (k, e, cos)


@pytest.mark.gpu
@pytest.mark.parametrize("engine", ["hip", "torch"])
def test_gpu_trainer_learns_from_a_teacher(tmp_path, engine):
    data = np.random.default_rng(0).integers(0, 12, (96, 32))
    torch.manual_seed(7)
    hist = T.train("kd", _model(2), data, None, str(tmp_path), batch_size=32, max_steps=6, device="cuda", log=lambda *a: None,
                   demo_every=0, engine=engine, teacher=_model(1), teacher_top_k=4)
    assert len(hist) == 6 and np.isfinite(hist).all()


def _changes(m):
    """What changes a model's weights or statistics, one after the other."""
    other = _model(5).to(next(m.parameters()).device)
    yield "load_state_dict", lambda: m.load_state_dict(other.state_dict())
    x = torch.randint(0, 12, (16, 32), generator=torch.Generator().manual_seed(2)).to(next(m.parameters()).device)

    def optimizer_step():
        m.train()
        opt = torch.optim.Adam(m.parameters(), lr=0.05)
        m.compute_loss(x, 0.3, 0.05)["loss"].backward()
        opt.step()

    def statistics_alone():
        m.train()
        with torch.no_grad():
            m.compute_loss(x, 0.3, 0.05)

    def reassigned():
        with torch.no_grad():
            for _ in range(3):                        # a freed weight's address may come back
                m.generative_net.dense.weight = torch.nn.Parameter(torch.randn_like(m.generative_net.dense.weight) * 0.2)
                m.inference_net.dense.weight.data = torch.randn_like(m.inference_net.dense.weight) * 0.2

    yield "optimizer step", optimizer_step
    yield "moving statistics", statistics_alone
    yield "reassigned", reassigned


def test_folded_weights_know_what_they_were_made_from():
    """Copies of weights in the kernels' layouts are stale after any change of what they were made from."""
    from serann.ops.riboae_ops import HipRiboDecoder, HipRiboEncoder
    m = _model(1)
    for name, change in _changes(m):
        dec, enc = HipRiboDecoder(m, "cpu"), HipRiboEncoder(m, "cpu")
        m.eval()
        m.encode_tokens(np.zeros((2, 32), np.int64))
        assert not dec.stale(m) and not enc.stale(m) and not dec.stale(m, "cpu") and dec.stale(m, "meta")
        change()
        assert dec.stale(m) and enc.stale(m), name
    dec = HipRiboDecoder(m, "cpu")
    assert dec.stale(copy.deepcopy(m))
    m._param_version = 7
    assert dec.stale(m)


@pytest.mark.gpu
def test_gpu_scores_and_targets_follow_the_weights():
    """Scores, teacher targets and codes are those of a model made anew from the current weights, whatever changed them."""
    from serann.riboae.hip_trainer import HipRiboTrainer
    m = _model(1).cuda()
    bits, x = _bits(9), torch.randint(0, 12, (9, 32), generator=torch.Generator().manual_seed(8)).cuda()

    def look(model):
        s = model.score_tokens(bits, device="cuda", top_k=3)
        ids, lp, _ = model.distill_targets(x, 4)
        return [s[k] for k in sorted(s)] + [ids.cpu().numpy(), lp.cpu().numpy(), model.encode_tokens(x.cpu().numpy(), "cuda"),
                                            model.decode_tokens(bits, "cuda")]

    def agree(name):
        fresh = _model(3).cuda()
        fresh.load_state_dict(m.state_dict())
        for a, b in zip(look(m), look(fresh)):
            np.testing.assert_array_equal(a, b, err_msg=name)

    before = look(m)
    for name, change in _changes(m):
        change()
        agree(name)
        after = look(m)
        assert any((a != b).any() for a, b in zip(before, after)), name
        before = after
    tr = HipRiboTrainer(m.train(), device="cuda")
    tr.step(x, 0.3, 0.05, 0.05)
    agree("trainer step")
    tr.step(x, 0.3, 0.05, 0.05, update=False)
    agree("step without update")


def test_folded_weights_stay_with_their_model():
    import pickle
    from serann.ops.riboae_ops import HipRiboDecoder
    m = _model(1)
    m._hip_decoder = HipRiboDecoder(m, "cpu")
    assert copy.deepcopy(m)._hip_decoder is None and pickle.loads(pickle.dumps(m))._hip_decoder is None
    assert m._hip_decoder is not None


@pytest.mark.gpu
def test_gpu_targets_and_scores_from_two_streams_and_two_threads():
    """Batches of one size share a model's buffers: calls from other streams and threads come out as one after the other."""
    import threading
    m = _model(1).cuda()
    g = torch.Generator().manual_seed(4)
    xs = [torch.randint(0, 12, (24, 32), generator=g).cuda() for _ in range(6)]
    bits = [_bits(24, seed=s) for s in range(6)]
    want = [m.distill_targets(x, 4)[:2] for x in xs]
    scored = [m.score_tokens(b, device="cuda", top_k=2) for b in bits]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(4):                                # one thread, no waits between the streams
        got = []
        for i, x in enumerate(xs):
            with torch.cuda.stream(streams[i % 3]):
                got.append(m.distill_targets(x, 4)[:2])
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    out, errors = {}, []

    def work(k):
        try:
            with torch.cuda.stream(streams[k]):
                for i in range(6):
                    out[k, i] = m.distill_targets(xs[i], 4)[:2] + (m.score_tokens(bits[i], device="cuda", top_k=2),)
                torch.cuda.current_stream().synchronize()
        except BaseException as e:                    # a failed thread is a failed test
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(3)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not errors, errors
    for (_, i), (ids, lp, s) in out.items():
        assert torch.equal(ids, want[i][0]) and torch.equal(lp, want[i][1])
        for k in s:
            np.testing.assert_array_equal(s[k], scored[i][k])


@pytest.mark.gpu
def test_a_refused_teacher_leaves_the_hip_trainer_as_it_was():
    from serann.riboae.hip_trainer import HipRiboTrainer
    m = _model(2).cuda().train()
    tr = HipRiboTrainer(m, device="cuda")
    x = torch.randint(0, 12, (16, 32), generator=torch.Generator().manual_seed(1)).cuda()
    ids, lp, t = _model(1).cuda().distill_targets(x, 4)
    tr.step(x, 0.3, 0.05, 1e-3, teacher=(ids, lp, t))
    torch.cuda.synchronize()
    was = [v.clone() for v in (tr.p, tr.stats, tr.m, tr.v, tr.step_i)]
    for bad in ((ids.cpu(), lp, t), (ids[:8], lp[:8], t), (ids.float(), lp, t), (ids, lp, 0.0), (ids, lp), (ids, lp[..., :2], t)):
        with pytest.raises((TypeError, ValueError)):
            tr.step(x, 0.3, 0.05, 1e-3, teacher=bad)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(was, (tr.p, tr.stats, tr.m, tr.v, tr.step_i)))
    tr.step(x, 0.3, 0.05, 1e-3, teacher=(ids, lp, t))
    assert int(tr.step_i) == int(was[4]) + 1


@pytest.mark.gpu
def test_gpu_scores_and_targets_in_and_after_inference_mode():
    """What a model keeps for the kernels is of use in inference mode and outside, whichever asked first."""
    bits, x = _bits(7), torch.randint(0, 12, (7, 32), generator=torch.Generator().manual_seed(3)).cuda()

    def look(m):
        s = m.score_tokens(bits, device="cuda", top_k=3)
        ids, lp, _ = m.distill_targets(x, 4)
        return [s[k] for k in sorted(s)] + [ids.cpu().numpy(), lp.cpu().numpy(), m.encode_tokens(x.cpu().numpy(), "cuda")]

    want = look(_model(1).cuda())
    m = _model(1).cuda()
    with torch.inference_mode():
        inside = look(m)
    after = look(m)
    with torch.inference_mode():
        again = look(m)
        made_inside = look(_model(1).cuda())
    for got in (inside, after, again, made_inside):
        for a, b in zip(got, want):
            np.testing.assert_array_equal(a, b)
