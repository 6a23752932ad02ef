"""The engine's layer chains with norm, dropout and labels (mmvae_cfg.layer_norm / dropout / n_labels)
against the oracle models with the same layers (oracle/layers.py), on the GPU: losses, every registered
gradient, the optimiser, the recorder's encode; step graphs, poisoned workspaces, streamed data,
data-parallel shards, the command line.  Tolerances: the wide path's (loss 2e-5, gradients 2e-4
norm-relative: f32 and bf16x3 against the f32 oracle)."""
import gzip
import os
import subprocess

import numpy as np
import pytest
import torch

import mmvae_amd
from helpers import assert_adam_close, assert_grads_close, rel_err
from mmvae_amd import MODEL_NB, MODEL_VMF, Engine, MMVAEError, host
from oracle import layers, nb_oracle, synth, vmf_oracle
from oracle.adam import LibTorchAdam, clip_grad_norm_

pytestmark = pytest.mark.gpu
SEED = 11


def labels_for(N, V, seed=0):
    lab = np.random.default_rng(seed).integers(0, V, N).astype(np.int32)
    lab[::17] = -1
    return lab


def engine(model, dtype, D=700, K=24, B=96, N=400, V=5, seed=SEED, **kw):
    eng = Engine(D=D, K=K, max_batch=B, dtype=dtype, seed=seed, model=MODEL_VMF if model == "vmf" else MODEL_NB, n_labels=V, **kw)
    assert eng.path() == "wide"
    eng.synth_csr(N, lib_size=1200.0, seed=3)
    if V:
        eng.set_labels(labels_for(N, V))
    eng.init_params(seed=7)
    if model == "vmf":
        eng.set_param("ln_kappa", np.array([np.log(np.float32(4.0))], np.float32))
    rng = np.random.default_rng(3)
    for n, k, _ in eng.param_info():  # weights away from 1 and 0, so that their places matter
        if ".norm_" in n:
            eng.set_param(n, (1.0 if n.endswith("weight") else 0.0) + 0.3 * rng.standard_normal(k))
    return eng


def oracle_of(eng, model, enc, dec, relu, **kw):
    shape = {n: k for n, k, _ in eng.param_info()}
    if model == "vmf":
        p0, f0 = vmf_oracle.init_params(eng.D, Z=eng.K, enc_layers=enc, dec_layers=dec)
    else:
        p0, f0 = nb_oracle.init_params(eng.D, K=eng.K, enc_layers=enc, dec_layers=dec, relu=relu)
    pull = lambda d: {n: torch.from_numpy(eng.get_param(n, shape[n]).reshape(v.shape)) for n, v in d.items()}  # noqa: E731
    p = pull(p0)
    for n, k, reg in eng.param_info():
        if reg and n not in p:
            p[n] = torch.from_numpy(eng.get_param(n, k))
            if n == "label_embedding.weight":
                p[n] = p[n].view(-1, eng.K)
    m = (layers.VMFLayers if model == "vmf" else layers.NBLayers)(p, pull(f0), relu=relu)
    for k, v in kw.items():
        setattr(m, k, v)
    return m


CASES = [
    ("nb", "f32", (40, 130), (33, 20), False, True, 0.2, 5),
    ("nb", "bf16x3", (40, 130), (33,), False, True, 0.2, 5),
    ("nb", "bf16x3", (), (64,), True, True, 0.0, 0),
    ("nb", "f32", (), (), False, False, 0.3, 3),
    ("nb", "bf16x3", (50,), (), False, False, 0.0, 1),
    ("nb", "f32", (), (48, 48), True, False, 0.25, 0),
    ("vmf", "f32", (40, 130), (33, 20), True, True, 0.2, 5),
    ("vmf", "bf16x3", (90,), (70,), True, False, 0.1, 4),
    ("vmf", "f32", (), (), False, True, 0.0, 7),
]


@pytest.mark.parametrize("model,dtype,enc,dec,relu,norm,p,V", CASES)
def test_layers_follow_the_oracle(model, dtype, enc, dec, relu, norm, p, V):
    B, beta, N = 96, 0.7, 400
    eng = engine(model, dtype, V=V, layer_norm=norm, dropout=p, label_scale=1.5, relu=relu, enc_hidden=enc, dec_hidden=dec)
    m = oracle_of(eng, model, enc, dec, relu, layer_norm=norm, dropout=p, label_scale=1.5)
    adam = LibTorchAdam(m.registered() if model == "nb" else list(m.p.values()), lr=1e-3, weight_decay=1e-4)
    lab = labels_for(N, V) if V else None
    rng = np.random.default_rng(5)
    for t in range(3):
        b = B if t != 1 else 61
        cells = (np.arange(b, dtype=np.int64) * 7 + 11 * t) % N
        if t == 2:
            cells[5] = cells[4]  # the same cell twice
        em, en = rng.standard_normal((b, eng.K)).astype(np.float32), rng.standard_normal((b, 1)).astype(np.float32)
        rp, col, val = eng.get_rows(cells)
        x, c = torch.from_numpy(synth.densify(rp, col, val, np.arange(b), eng.D)), torch.ones(b, 1)
        step = 2 ** 33 + t
        m.key = (SEED, step, 64)
        m.labels = torch.from_numpy(lab[cells]).long() if V else None

        def loss_of():
            if model == "vmf":
                return vmf_oracle.vmf_vae_loss(x, m.forward(x, c, torch.from_numpy(em)), beta)
            return nb_oracle.loss(x, m.forward(x, c, torch.from_numpy(em), torch.from_numpy(en)), beta)
        eps = em.ravel() if model == "vmf" else np.concatenate([em.ravel(), en.ravel()])
        L = loss_of()
        got = eng.run(cells, beta, eps=eps, update=False, step_id=step, row_offset=64)[0]
        assert abs(got - float(L.detach())) <= 2e-5 * abs(float(L.detach())), (t, got, float(L.detach()))
        loss, total = eng.step(cells, beta, eps=eps, step_id=step, row_offset=64)
        assert abs(loss - float(L.detach())) <= 2e-5 * abs(float(L.detach()))
        adam.zero_grad()
        L.backward()
        gold = {k: v.grad.detach().numpy().copy() for k, v in m.p.items()}
        grads = eng.grads()
        assert set(grads) == set(gold)
        if model == "vmf":  # fp32 cancellation of df/kappa-sized terms
            gk, wk = float(grads["ln_kappa"][0]), float(gold["ln_kappa"][0])
            assert abs(gk - wk) <= 1e-6 * (0.5 * eng.D - 1.0) + 2e-4 * abs(wk), (gk, wk)
        assert_grads_close(grads, {k: v for k, v in gold.items() if k != "ln_kappa"}, 2e-4, ctx=f"step {t}")
        want_total = clip_grad_norm_([v.grad for v in m.p.values()], 1.0)
        assert abs(total - want_total) <= 2e-3 * want_total
        adam.step()
        params = {k: v.detach().numpy().copy() for k, v in m.p.items()}
        assert_adam_close(eng.params(registered_only=True), params, gold, ctx=f"step {t}", noisy_keys=("ln_kappa",) if model == "vmf" else ())
        eng.set_params(params)  # (the next step from the same place)
    m.training = False
    mean, lv = eng.encode(cells)
    with torch.no_grad():
        wm, wlv = m.encode_mu(x) if model == "nb" else m.encode(x)
    assert rel_err(mean, wm.numpy()) < 2e-5 and rel_err(lv, wlv.numpy()) < 2e-5


def test_parameters_behind_the_references():
    """The reference's parameters keep their names, order and initial values; the layers' come behind them, weights 1, biases 0."""
    kw = dict(D=60, K=8, max_batch=32, dtype="f32", enc_hidden=(10,), dec_hidden=(12, 9))
    plain, with_ = Engine(**kw), Engine(layer_norm=True, dropout=0.1, n_labels=4, **kw)
    for e in (plain, with_):
        e.init_params(seed=3)
    a, b = plain.param_info(), with_.param_info()
    assert b[:len(a)] == a
    assert [n for n, _, r in b[len(a):] if r] == ["mu_enc.norm_1.weight", "mu_enc.norm_1.bias", "mu_dec.norm_1.weight", "mu_dec.norm_1.bias",
                                                  "mu_dec.norm_2.weight", "mu_dec.norm_2.bias", "label_embedding.weight"]
    pa, pb = plain.params(), with_.params()
    for n in pa:
        assert np.array_equal(pa[n], pb[n]), n
    assert (pb["mu_enc.norm_1.weight"] == 1).all() and not pb["mu_dec.norm_2.bias"].any()
    assert 0 < np.abs(pb["label_embedding.weight"]).max() <= 8 ** -0.5


@pytest.mark.parametrize("model", ["nb", "vmf"])
def test_graph_equals_eager_under_poison(model):
    """Replayed step graphs (labels, dropout keys and noise change from step to step) equal eager steps to the bit,
    whatever the workspaces held."""
    res = []
    for graph in (False, True):
        eng = engine(model, "bf16x3", V=6, layer_norm=True, dropout=0.2, enc_hidden=(40,), dec_hidden=(50,), relu=model == "vmf")
        eng.graph(graph)
        out = []
        for s, b in enumerate([96, 50, 96, 96, 50]):
            if graph:
                eng.poison(0xFF)
            out.append(eng.step((np.arange(b, dtype=np.int64) * 3 + 17 * s) % 400, 0.6, step_id=s))
            if s == 2:
                eng.set_labels(labels_for(400, 6, seed=9))
        out.append(eng.eval_loss(np.arange(96, dtype=np.int64), 0.6, step_id=9))
        if graph:
            assert eng.graph_stats()["replays"] >= 6
        res.append((out, eng.params(registered_only=True)))
    assert res[0][0] == res[1][0]
    for k in res[0][1]:
        assert np.array_equal(res[0][1][k], res[1][1][k]), k


def test_streamed_equals_resident():
    rng = np.random.default_rng(0)
    N, D = 300, 200
    x = rng.poisson(0.5, (N, D)).astype(np.float32)
    rowptr = np.concatenate([[0], np.cumsum((x > 0).sum(1))]).astype(np.int64)
    col, val = np.nonzero(x)[1].astype(np.int32), x[x > 0]
    out = []
    for stream in (False, True):
        eng = Engine(D=D, K=16, max_batch=64, dtype="bf16x3", layer_norm=True, dropout=0.1, n_labels=9, dec_hidden=(32,))
        (eng.stream_csr if stream else eng.upload_csr)(rowptr, col, val)
        eng.set_labels(labels_for(N, 9))
        eng.init_params(seed=1)
        out.append([eng.step((np.arange(64) * 11 + s) % N, 0.5, step_id=s) for s in range(4)] + [eng.params()])
    assert out[0][:4] == out[1][:4]
    for k in out[0][4]:
        assert np.array_equal(out[0][4][k], out[1][4][k]), k


@pytest.mark.parametrize("model", ["nb", "vmf"])
def test_shards_sum_to_the_whole_batch(model):
    """Data-parallel shards (local decomposition): masks by global row, labels by cell; gradients sum to the whole batch's."""
    B, world = 96, 3
    cells = (np.arange(B, dtype=np.int64) * 5 + 3) % 400
    kw = dict(V=5, layer_norm=True, dropout=0.3, enc_hidden=(40,), dec_hidden=(30,))
    full = engine(model, "f32", **kw)
    l_full, _ = full.step(cells, 0.7, step_id=5)
    want, b = full.grads(), B // world
    tot, gsum = 0.0, None
    for r in range(world):
        eng = engine(model, "f32", B=b, **kw)
        eng.comm_init(r, world, None)
        tot += eng.step(cells[r * b:(r + 1) * b], 0.7, n_total=B, row_offset=r * b, step_id=5)[0]
        g = eng.grads()
        gsum = g if gsum is None else {k: gsum[k] + g[k] for k in g}
    assert abs(tot - l_full) <= 2e-5 * abs(l_full)
    for k in want:
        if k == "ln_kappa":
            assert abs(float(gsum[k][0] - want[k][0])) <= 1e-6 * (0.5 * full.D - 1.0)
            continue
        assert rel_err(gsum[k], want[k]) <= 2e-5, (k, rel_err(gsum[k], want[k]))


def test_label_refusals_and_states():
    eng = Engine(D=60, K=8, max_batch=32, n_labels=3)
    with pytest.raises(MMVAEError, match="no dataset"):
        eng.set_labels([0])
    eng.synth_csr(50, lib_size=100.0)
    eng.init_params(seed=1)
    cells = np.arange(20)
    with pytest.raises(MMVAEError, match="labels are not set"):
        eng.step(cells, 1.0)
    eng.encode(cells)  # (reads no labels)
    for bad, msg in (([0] * 49, "number of cells"), ([3] * 50, "label 3"), ([-2] * 50, "label -2"), ([0.5] * 50, "whole numbers"), ([2 ** 40] * 50, "whole")):
        with pytest.raises(MMVAEError, match=msg):
            eng.set_labels(bad)
    eng.set_labels([-1] * 50)  # nobody has a label
    eng.step(cells, 1.0)
    assert not eng.get_grad("label_embedding.weight", 24).any()
    eng.synth_csr(50, lib_size=100.0)  # a new dataset forgets them
    with pytest.raises(MMVAEError, match="labels are not set"):
        eng.step(cells, 1.0)
    with pytest.raises(MMVAEError, match="has no labels"):
        e2 = Engine(D=60, K=8, max_batch=32)
        e2.synth_csr(50, lib_size=100.0)
        e2.set_labels([0] * 50)


@pytest.mark.parametrize("V", [5, 90])
def test_small_batches_on_a_handle_for_large_ones(V):
    """A batch of 20,000 and one of 32,768 on a handle for 40,000 (which has fewer, longer pieces of a label's tokens than
    they have) give what a handle of their own size gives."""
    kw = dict(D=70, V=V, enc_hidden=(12,), dec_hidden=(16,), layer_norm=True)
    big = engine("nb", "f32", B=40000, **kw)
    start = big.params(registered_only=True)
    for B in (20000, 32768, 40000):
        own = engine("nb", "f32", B=B, **kw)
        cells = (np.arange(B, dtype=np.int64) * 7) % 400
        eps = np.random.default_rng(B).standard_normal(B * (big.K + 1)).astype(np.float32)
        big.set_params(start)
        a, b = (e.step(cells, 0.7, eps=eps, step_id=3)[0] for e in (big, own))
        assert abs(a - b) <= 2e-5 * abs(b), B
        assert_grads_close(big.grads(), own.grads(), 2e-4, ctx=f"batch {B}")


def test_dropout_draws_new_masks_each_step_and_none_in_encode():
    eng = engine("nb", "f32", V=0, dropout=0.5)
    cells, zero = np.arange(96), np.zeros(96 * (eng.K + 1), np.float32)
    a = [eng.run(cells, 0.5, eps=zero, update=False, step_id=s)[0] for s in (1, 2, 1)]
    assert a[0] == a[2] and a[0] != a[1]
    m = [eng.encode(cells)[0] for _ in range(2)]
    assert np.array_equal(m[0], m[1])


@pytest.mark.parametrize("exe", ["nb_vae_main", "vmf_vae_main"])
def test_command_line(tmp_path, exe):
    """--layer_norm --dropout --labels --label_scale end to end: finite scores, the layers' parameters recorded."""
    N, D = 120, 80
    x = np.random.default_rng(1).poisson(0.6, (N, D))
    x[:, 0] += 1
    lines = [f"{g + 1} {c + 1} {x[c, g]}" for c in range(N) for g in range(D) if x[c, g]]
    mtx = tmp_path / "x.mtx.gz"
    with gzip.open(mtx, "wt") as f:
        f.write("%%MatrixMarket matrix coordinate integer general\n" + f"{D} {N} {len(lines)}\n" + "\n".join(lines) + "\n")
    lab = tmp_path / "labels.txt.gz"
    with gzip.open(lab, "wt") as f:
        f.write("\n".join("NA" if i % 10 == 0 else str(i % 4) for i in range(N)) + "\n")
    hidden = ["--mean_encoding", "24", "--mean_decoding", "20"] if exe == "nb_vae_main" else ["--encoding", "24", "--decoding", "20"]
    out = tmp_path / "o"
    r = subprocess.run([os.path.join(host.BIN_DIR, exe), "--mtx", str(mtx), "--out", str(out), "--batch_size", "40", "--max_epoch", "4", "--recording", "2",
                        "--layer_norm", "--dropout", "0.1", "--labels", str(lab), "--label_scale", "0.5", *hidden],
                       capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stderr
    scores = np.loadtxt(str(out) + ".scores.gz")
    assert scores.shape == (4,) and np.isfinite(scores).all()
    s = "mu" if exe == "nb_vae_main" else "z"
    files = os.listdir(tmp_path)
    for name in (f"{s}_enc.norm_1.weight", f"{s}_dec.norm_1.bias", "label_embedding.weight"):
        assert any(name in f for f in files), (name, files)
    emb = next(f for f in files if "label_embedding.weight" in f)
    assert np.loadtxt(tmp_path / emb).shape == (4, 2)
