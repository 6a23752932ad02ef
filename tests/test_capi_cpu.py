"""CPU tests of the C-ABI library: it loads, exports every symbol include/mmvae_capi.h
declares, and the host-only entry points (operators.hh scalars, cfg defaults, graceful
failure without a GPU) behave — no compute calls."""
import ctypes
import os
import re
import subprocess

import numpy as np
import pytest

import mmvae_amd
from oracle import fastmath


def declared_functions():
    src = open(mmvae_amd.HEADER_PATH).read()
    src = re.sub(r"/\*.*?\*/", "", src, flags=re.S)
    return sorted(set(re.findall(r"\b(mmvae_[a-z0-9_]+)\s*\(", src)))


def test_library_exports_every_declared_symbol():
    L = ctypes.CDLL(mmvae_amd.LIB_PATH)
    names = declared_functions()
    assert len(names) >= 25
    missing = [n for n in names if not hasattr(L, n)]
    assert not missing, missing


def test_binding_covers_header():
    mmvae_amd.lib()  # sets every signature; raises on a missing symbol


def test_cfg_defaults_match_reference():
    c = mmvae_amd.default_cfg(mmvae_amd.MODEL_NB)
    assert c.K == 2 and c.H == 1 and c.R == 1 and c.max_batch == 100      # nb.hh:59-61, mmvae.hh:35
    assert abs(c.lr - 1e-3) < 1e-9 and abs(c.weight_decay - 1e-4) < 1e-9  # mmvae_alg.hh:19,236
    assert c.grad_clip == 1.0                                              # Q7
    assert abs(c.kappa_min - 0.1) < 1e-7 and c.kappa_max == 10.0          # vmf.hh:61-62


def test_host_fastmath_bit_exact():
    xs = np.random.default_rng(1).uniform(1e-3, 3e4, 500).astype(np.float32)
    for x in list(xs) + [np.float32(2 * np.pi), np.float32(25.0)]:
        assert np.float32(mmvae_amd.fasterlog(float(x))) == fastmath.fasterlog(x)
        assert np.float32(mmvae_amd.fasterlgamma(float(x))) == fastmath.fasterlgamma(x)


def test_lbessel_matches_oracle_and_q3():
    import torch
    from oracle.vmf_oracle import lbessel_op
    for kappa, nu in [(5.0, 24.0), (0.1, 9999.0), (30.0, 4.0), (2.0, 2.0)]:
        got = mmvae_amd.lbessel(kappa, nu)
        k = torch.tensor([kappa], dtype=torch.float32, requires_grad=True)
        want = lbessel_op(k, nu)
        assert abs(got - want.item()) <= 2e-6 * max(1.0, abs(want.item())), (kappa, nu, got, want.item())
        want.backward(torch.tensor([-3.0]))  # Q3: upstream ignored
        assert abs(mmvae_amd.lbessel_grad(kappa, nu) - float(k.grad)) <= 1e-6 * abs(float(k.grad))
    assert abs(mmvae_amd.lbessel_grad(5.0, 24.0) - 4.901020) < 1e-5  # SURVEY Q3 probe


def test_create_without_gpu_fails_cleanly():
    import torch
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    with pytest.raises(mmvae_amd.MMVAEError):
        mmvae_amd.Engine(D=10, K=2)


@pytest.mark.parametrize("kw,msg", [
    # nb.hh:334-337: --relu with hidden --mean_encoding layers is the reference's construction error (Q2)
    (dict(relu=True, enc_hidden=(16,)), "mu_encoding_1"),
    (dict(enc_hidden=(0,)), "hidden encoder widths must be >= 1"),
    (dict(dec_hidden=(8, 0)), "hidden decoder widths must be >= 1"),
    (dict(enc_hidden=(8,) * 17), "at most 16"),
])
def test_hidden_layer_cfg_validated_before_any_device(kw, msg):
    """cfg checks of mmvae_create run before the device is touched: the same error here and on a GPU box."""
    with pytest.raises(mmvae_amd.MMVAEError, match=msg):
        mmvae_amd.Engine(D=10, K=4, **kw)


@pytest.mark.parametrize("kw,msg", [
    (dict(D=0, K=4), "need D, K, C, H, R, max_batch >= 1"),
    (dict(D=10, K=0), "need D, K, C, H, R, max_batch >= 1"),
    (dict(D=10, K=4, C=0), "need D, K, C, H, R, max_batch >= 1"),
])
def test_shape_limits_validated_before_any_device(kw, msg):
    """Invalid shapes are MMVAE_E_ARG at create time, before the device is touched.  Every valid
    shape is accepted: K, hidden widths, C / H / R and D beyond the fused kernels' envelope run on
    the wide path (mm-vae_amd/csrc/wide.hip), so e.g. D = 75,265 or K = 65 only fail here for the
    missing GPU."""
    with pytest.raises(mmvae_amd.MMVAEError, match=msg):
        mmvae_amd.Engine(**kw)


@pytest.mark.parametrize("kw", [dict(D=75265, K=4), dict(D=10, K=128), dict(D=10, K=4, C=12, H=9, R=10),
                                dict(D=10, K=4, enc_hidden=(256, 128), dec_hidden=(8,) * 16)])
def test_wide_shapes_accepted(kw):
    """Shapes the reference trains (any latent / hidden width, nb.hh:331-379, vmf.hh:338-385) pass
    the cfg checks: without a GPU the only error is the missing device."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    with pytest.raises(mmvae_amd.MMVAEError, match="no HIP device"):
        mmvae_amd.Engine(**kw)


GRAPH_KEY_PROBE = r"""
#include "graph_key.hpp"
#include <cstdio>
#include <cstdlib>
#include <random>
using namespace mmvae;
// argv: world n_total comm_graph no_balance_mask(per rank bits) seed
int main(int argc, char** argv) {
    const int world = atoi(argv[1]);
    const long n_total = atol(argv[2]);
    const bool comm_graph = atoi(argv[3]) != 0;
    const int nb_mask = atoi(argv[4]);
    std::mt19937 rng(atoi(argv[5]));
    // comm_sync_capacity: MMVAE_NO_BALANCE max-agreed over the ranks
    bool no_balance = false;
    for (int r = 0; r < world; ++r) no_balance = no_balance || ((nb_mask >> r) & 1);
    for (int r = 0; r < world; ++r) {
        // the rank's slice of the global batch (trainer.cc / bench.py: B = n_total / world, the
        // last rank taking any remainder) and a rank-local batch: its own cells and nonzero counts
        const long B = r < world - 1 ? n_total / world : n_total - (world - 1) * (n_total / world);
        long nnz = 0;
        for (long j = 0; j < B; ++j) nnz += rng() % 4000;
        KeyInputs in;
        in.B = B;
        in.n_total = n_total;
        in.beta = 0.5f;
        in.update = true;
        in.world = world;
        in.comm_graph = comm_graph;
        in.perm = balance_rule(B, false, true, no_balance);
        in.ents = (const void*)(0x1000 + 64 * r);  // a rank-local device pointer
        in.gen = 3;
        GraphKey k;
        const int rc = derive_graph_key(in, &k);
        int64_t w[6];
        key_words(k, w);
        printf("%d %d", r, rc);
        for (int i = 0; i < 6; ++i) printf(" %lld", (long long)w[i]);
        printf(" %ld\n", nnz);
    }
    return 0;
}
"""


@pytest.fixture(scope="module")
def graph_key_probe(tmp_path_factory):
    import subprocess
    d = tmp_path_factory.mktemp("gk")
    src = d / "probe.cc"
    src.write_text(GRAPH_KEY_PROBE)
    exe = d / "probe"
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mm-vae_amd", "csrc")
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", csrc, str(src), "-o", str(exe)], check=True)

    def run(world, n_total, comm_graph, nb_mask=0, seed=1):
        out = subprocess.run([str(exe), str(world), str(n_total), str(int(comm_graph)), str(nb_mask), str(seed)],
                             check=True, capture_output=True, text=True).stdout
        return [tuple(int(v) for v in line.split()) for line in out.strip().splitlines()]
    return run


@pytest.mark.parametrize("world", [2, 4, 8])
def test_graph_key_rank_invariant_under_differing_batches(graph_key_probe, world):
    """VERDICT r5 item 7 (capi.hip mmvae_run, graph_key.hpp): with RCCL calls inside step graphs
    every rank must derive the same key words at every step, whatever rows and nonzero counts its
    own batch holds, so all ranks capture (and run the capture agreement) at the same steps."""
    for seed in range(3):
        rows = graph_key_probe(world, 4096 * world, True, seed=seed)
        assert all(r[1] == 0 for r in rows)
        assert len({r[2:8] for r in rows}) == 1, rows          # identical key words
        assert len({r[8] for r in rows}) == world              # from different batches
        # MMVAE_NO_BALANCE set on one rank only: agreed (max) before the rule, still one key
        rows = graph_key_probe(world, 4096 * world, True, nb_mask=1 << (world - 1), seed=seed)
        assert len({r[2:8] for r in rows}) == 1 and (rows[0][5] >> 2) & 1 == 0, rows


@pytest.mark.parametrize("world", [2, 3, 8])
def test_graph_key_uneven_slices_refused_before_any_collective(graph_key_probe, world):
    """Uneven slices (n_total % world != 0) would give the ranks different B — and B % 16 decides
    the permutation flag — so their keys could diverge and one rank would capture alone.  The key
    derivation refuses it on the ranks whose slice differs (a rank-local MMVAE_E_ARG before the
    step issues any collective), and eager steps (no comm graph) are unaffected."""
    n_total = 4096 * world + 1
    rows = graph_key_probe(world, n_total, True)
    assert any(r[1] == -1 for r in rows), rows
    assert all(r[1] == -1 or r[2] * world == n_total for r in rows)
    assert all(r[1] == 0 for r in graph_key_probe(world, n_total, False))


OLDER_CLIENT = r"""
#include <stdint.h>
#include <stdio.h>
#include <string.h>
struct cfg {  /* mmvae_cfg as it was before the layer options */
    int32_t model, dtype;
    int64_t D, C, K, H, R, max_batch;
    float lr, weight_decay, grad_clip, kappa_min, kappa_max;
    uint64_t seed;
    int32_t relu, n_enc_hidden, n_dec_hidden, enc_hidden[16], dec_hidden[16];
};
void mmvae_cfg_default(struct cfg*, int32_t);
int mmvae_create(const struct cfg*, int, void**);
const char* mmvae_last_error(void*);
int main(void) {
    struct { struct cfg c; unsigned char behind[64]; } s;
    void* h;
    int i, touched = 0;
    memset(&s, 0xff, sizeof(s));  /* (as floats: NaN, which the layer options refuse) */
    mmvae_cfg_default(&s.c, 0);
    for (i = 0; i < 64; ++i) touched += s.behind[i] != 0xff;
    s.c.D = 10;
    i = mmvae_create(&s.c, 99, &h);
    printf("%d %d %d %g|%s\n", touched, i, (int)s.c.max_batch, s.c.kappa_max, mmvae_last_error(0));
    memset((char*)&s.c + 76, 0xff, 4);  /* a cfg filled by hand: its padding holds anything */
    i = mmvae_create(&s.c, 99, &h);
    printf("%d|%s\n", i, mmvae_last_error(0));
    return 0;
}
"""


def test_programs_built_before_the_layer_options(tmp_path):
    """Their cfg ends at dec_hidden: nothing behind it is written or read."""
    c = tmp_path / "older.c"
    c.write_text(OLDER_CLIENT)
    subprocess.run(["gcc", str(c), "-o", str(tmp_path / "older"), mmvae_amd.LIB_PATH, "-Wl,-rpath," + os.path.dirname(mmvae_amd.LIB_PATH),
                    "-Wl,--allow-shlib-undefined"], check=True)
    out = subprocess.run([str(tmp_path / "older")], check=True, capture_output=True, text=True).stdout.splitlines()
    assert out == ["0 -2 100 10|no HIP device 99", "-2|no HIP device 99"]


def test_cfg_carries_its_size():
    """Through the header and the binding a cfg holds its size, and the layer options count."""
    c = mmvae_amd.default_cfg(mmvae_amd.MODEL_NB)
    assert c.size == ctypes.sizeof(c) and c.label_scale == 1.0
    assert mmvae_amd.Cfg().size == ctypes.sizeof(c)  # (one filled by hand too)
    h, L = ctypes.c_void_p(), mmvae_amd.lib()
    c.D, c.dropout = 10, 2.0
    assert L.mmvae_create(ctypes.byref(c), 99, ctypes.byref(h)) == -1 and b"dropout" in L.mmvae_last_error(None)
    c.dropout, c.n_labels = 0.5, -1
    assert L.mmvae_create(ctypes.byref(c), 99, ctypes.byref(h)) == -1 and b"n_labels" in L.mmvae_last_error(None)
