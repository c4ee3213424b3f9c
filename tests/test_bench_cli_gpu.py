"""The command-line benchmark with the reference's flags (benchmark/bench_vanilla_spmm.py:71-84,
bench_vanilla_sddmm.py:77-90): ``--dataset <scipy npz> --feat-len F --target cuda``.  The
files are written as the reference's download script writes them
(benchmark/download_reddit_dataset.py:11-20): a canonical float32 CSR for SpMM, its COO
form for SDDMM.  The result the CLI computed is dumped and compared with the CPU oracle."""
import numpy as np
import pytest
import scipy.sparse as sp

from featgraph_b200 import bench_cli, graphs
from helpers import bits, random_csr

pytestmark = pytest.mark.gpu


def _files(tmp_path):
    csr = random_csr(700, 700, 0.05, seed=51, empty_rows=(0, 9), dense_rows=(33,))
    assert csr.has_canonical_format and csr.dtype == np.float32
    csr_path, coo_path = str(tmp_path / "adj_csr_float32.npz"), str(tmp_path / "adj_coo.npz")
    sp.save_npz(csr_path, csr)
    sp.save_npz(coo_path, csr.tocoo())
    return csr, csr_path, coo_path


def test_spmm_from_an_npz_file(tmp_path, oracle):
    csr, csr_path, _ = _files(tmp_path)
    dump = str(tmp_path / "y.npy")
    recs = bench_cli.main(["--kernel", "spmm", "--dataset", csr_path, "--feat-len", "64",
                           "--target", "cuda", "--num-runs", "3", "--dump-output", dump])
    assert len(recs) == 1 and recs[0]["nnz"] == csr.nnz and recs[0]["ms"] > 0
    assert recs[0]["graph"] == "file:" + csr_path and recs[0]["feat_len"] == 64
    x = graphs.normal_features(700, 64, graphs.FEAT_SEED, "cuda").cpu().numpy()
    want = oracle.spmm_csr_f32(csr.indptr, csr.indices, csr.data, x, n_cols=700)
    assert np.array_equal(bits(want), bits(np.load(dump)))


@pytest.mark.parametrize("heads", [1, 4])
def test_sddmm_from_an_npz_file_keeps_the_stored_edge_order(tmp_path, oracle, heads):
    csr, _, coo_path = _files(tmp_path)
    # a COO file whose edges are NOT in row-major order: the output follows the file
    coo = csr.tocoo()
    perm = np.random.default_rng(2).permutation(coo.nnz)
    shuffled = sp.coo_matrix((coo.data[perm], (coo.row[perm], coo.col[perm])), shape=coo.shape)
    sp.save_npz(coo_path, shuffled)
    dump = str(tmp_path / "out.npy")
    argv = ["--kernel", "sddmm", "--dataset", coo_path, "--target", "cuda", "--num-runs", "3",
            "--dump-output", dump]
    argv += ["--heads", "4", "--head-dim", "16"] if heads > 1 else ["--feat-len", "64"]
    recs = bench_cli.main(argv)
    assert recs[0]["nnz"] == coo.nnz and recs[0]["heads"] == heads
    shape = (4, 16) if heads > 1 else (64,)
    src = graphs.normal_features(700, shape, graphs.FEAT_SEED, "cuda").cpu().numpy()
    dst = graphs.normal_features(700, shape, graphs.FEAT2_SEED, "cuda").cpu().numpy()
    want = oracle.sddmm_coo_f32(shuffled.row, shuffled.col, src, dst, num_heads=heads)
    got = np.load(dump)
    assert np.array_equal(bits(want.reshape(got.shape)), bits(got))


@pytest.mark.parametrize("kernel, dtype", [("lookup", "bfloat16"), ("lookup-grad", "float32"),
                                           ("cross-entropy", "float16"), ("clip", "bfloat16"),
                                           ("train-step", "float32")])
def test_training_operators(kernel, dtype):
    recs = bench_cli.main(["--kernel", kernel, "--synthetic", "regular", "--vertices", "2048",
                           "--feat-len", "32,64", "--samples", "300", "--dtype", dtype,
                           "--num-runs", "2"])
    assert [r["feat_len"] for r in recs] == [32, 64] and all(r["ms"] > 0 for r in recs)
    assert recs[0]["kernel"] == kernel and recs[0]["vertices"] == 2048


def test_lookup_result_of_the_command(tmp_path):
    dump = str(tmp_path / "rows.npy")
    bench_cli.main(["--kernel", "lookup", "--synthetic", "regular", "--vertices", "500",
                    "--feat-len", "16", "--samples", "40", "--num-runs", "1", "--dump-output", dump])
    table = graphs.normal_features(500, 16, graphs.FEAT_SEED, "cuda")
    scaled = (table * np.float32(16 ** 0.5)).cpu().numpy()
    rows = np.load(dump)
    assert rows.shape == (40, 16)
    assert all((scaled == r).all(1).any() for r in rows)    # every row is a scaled row of the table


def test_train_step_is_refused_in_16_bits():
    with pytest.raises(SystemExit, match="float32"):
        bench_cli.main(["--kernel", "train-step", "--synthetic", "regular", "--vertices", "500",
                        "--feat-len", "16", "--dtype", "bfloat16"])


def test_the_x86_target_is_refused():
    with pytest.raises(SystemExit, match="cuda target only"):
        bench_cli.main(["--kernel", "spmm", "--synthetic", "regular", "--target", "x86"])
