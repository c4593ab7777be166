"""CPU-side checks: the C-ABI library loads and exports every symbol include/megacrn_hip.h declares,
the module surface matches the reference's state_dict layout / init RNG order, and the host logic
(curriculum draws, workspace sizing) behaves.  No compute calls (no GPU here)."""
import ctypes as C
import os
import re

import numpy as np
import pytest
import torch

from helpers import load_case

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_library_exports_every_declared_symbol():
    from megacrn_amd import _lib
    hdr = open(os.path.join(ROOT, "include", "megacrn_hip.h")).read()
    declared = set(re.findall(r"\b(mcrn_[a-z0-9_]+)\s*\(", hdr))
    assert declared, "no declarations parsed"
    lib = C.CDLL(_lib.LIB_PATH)
    missing = [s for s in sorted(declared) if not hasattr(lib, s)]
    assert not missing, missing
    assert set(_lib.EXPORTS) <= declared
    assert _lib.lib.mcrn_version() >= 100


def test_library_exports_only_the_c_abi():
    """-fvisibility=hidden (round 6): every exported FUNCTION is one the header declares; nothing of namespace mcrn's host code
    is in the dynamic symbol table (HIP's kernel-handle data objects are, by construction of the runtime's registration)."""
    import shutil
    import subprocess
    from megacrn_amd import _lib
    nm = shutil.which("nm")
    if not nm:
        pytest.skip("nm not present")
    hdr = open(os.path.join(ROOT, "include", "megacrn_hip.h")).read()
    declared = set(re.findall(r"\b(mcrn_[a-z0-9_]+)\s*\(", hdr))
    out = subprocess.run([nm, "-D", "--defined-only", _lib.LIB_PATH], capture_output=True, text=True, check=True).stdout
    funcs = {ln.split()[2] for ln in out.splitlines() if len(ln.split()) == 3 and ln.split()[1] in "TtWw"}
    funcs -= {"_init", "_fini"}
    exported_host_code = sorted(f for f in funcs if f.startswith("_Z"))
    assert not exported_host_code, exported_host_code[:5]
    assert {f for f in funcs if f.startswith("mcrn_")} == declared, sorted(declared ^ {f for f in funcs if f.startswith("mcrn_")})


def test_build_id_ties_measured_artefacts_to_the_library(tmp_path, monkeypatch):
    """the PMC traffic table bench.py reports must belong to the library that ran.  A table measured on
    another build (a deliberately stale file) makes `traffic` / `step_fabric_*` disappear; the newest profiles/r<NN>/ wins."""
    import json
    import bench
    from megacrn_amd import _lib
    bid = _lib.build_id()
    assert re.fullmatch(r"[0-9a-f]{16}", bid), bid
    prof = tmp_path / "profiles"
    (prof / "r7").mkdir(parents=True)
    (prof / "r12").mkdir()
    table = {"prop2_fwd_kernel<7, 2>": {"launches": 24, "hbm_bytes_per_launch_corrected": 3.0e7},
             "k_clip_adam": {"launches": 1, "hbm_bytes_per_launch_corrected": 1.0e6},
             "_step": {"fabric_bytes": 1.5e10, "dispatches": 358}}
    json.dump({**table, "_meta": {"build_id": bid, "git": "abc1234"}}, open(prof / "r7" / "traffic_metrla.json", "w"))
    monkeypatch.setattr(bench, "PROFILES_DIR", str(prof))
    d, src = bench.traffic_profile("metrla", "bf16x3")
    assert d is not None and src["status"] == "current" and src["file"].endswith("r7/traffic_metrla.json")
    assert bench.pmc_traffic("metrla", "bf16x3", 207) == 30000000
    st = bench.step_traffic("metrla", "bf16x3", 5.0)
    assert st["step_fabric_gb"] == 15.0 and st["step_fabric_tbs"] == 3.0 and st["traffic_source"]["status"] == "current"
    # a newer round's table from ANOTHER build: it is the newest, it is stale, nothing is reported (the older current one is not dug up)
    json.dump({**table, "_meta": {"build_id": "0" * 16}}, open(prof / "r12" / "traffic_metrla.json", "w"))
    d, src = bench.traffic_profile("metrla", "bf16x3")
    assert d is None and src["status"].startswith("stale") and "r12" in src["file"]
    assert bench.pmc_traffic("metrla", "bf16x3", 207) is None
    st = bench.step_traffic("metrla", "bf16x3", 5.0)
    assert "step_fabric_gb" not in st and st["traffic_source"]["status"].startswith("stale")
    # a table without a build id (the round-5 format) is stale too; no table at all says so
    json.dump(table, open(prof / "r12" / "traffic_metrla.json", "w"))
    assert bench.traffic_profile("metrla", "bf16x3")[0] is None
    assert bench.traffic_profile("pemsbay", "bf16x3")[1] == {"status": "absent"}
    # tile tables: same rule
    monkeypatch.setattr(bench, "TILE_DIR", str(tmp_path))
    json.dump({"build_id": "0" * 16, "words": []}, open(bench.tile_cache_path("syn8192", 32, "bf16"), "w"))
    assert not bench.tile_cache_current("syn8192", 32, "bf16") and not bench.import_tile_cache("syn8192", 32, "bf16")
    json.dump({"build_id": bid, "words": []}, open(bench.tile_cache_path("syn8192", 32, "bf16"), "w"))
    assert bench.tile_cache_current("syn8192", 32, "bf16") and bench.import_tile_cache("syn8192", 32, "bf16")


def test_traffic_table_of_the_current_build_stands_apart(tmp_path):
    """profiles/current/ holds the tables of the build at hand and goes before the dated ones, which stay what they were."""
    import json
    import bench
    prof = tmp_path / "profiles"
    for d, bid in (("r6", "a" * 16), ("r10", "b" * 16), ("current", "c" * 16)):
        (prof / d).mkdir(parents=True)
        json.dump({"_step": {"fabric_bytes": 1.0}, "_meta": {"build_id": bid}}, open(prof / d / "traffic_metrla.json", "w"))
    table, src = bench.traffic_profile("metrla", "bf16x3", str(prof), "c" * 16)
    assert table is not None and src["file"].endswith("current/traffic_metrla.json")
    assert bench.traffic_profile("metrla", "bf16x3", str(prof), "b" * 16)[0] is None
    (prof / "current" / "traffic_metrla.json").unlink()
    assert bench.traffic_profile("metrla", "bf16x3", str(prof), "b" * 16)[0] is not None


def test_flat_plane_sets_have_an_opt_out():
    """ADVICE (round 5): the per-cell gradient plane sets of the small graphs (ModelPlan::flat, up to 8 GB of workspace) can be switched
    off for smaller parts: MCRN_FLAT_SETS=0, read at plan time in a fresh process."""
    import subprocess
    import sys
    code = ("import ctypes as C, sys; sys.path.insert(0, %r); from megacrn_amd._lib import lib, Dims; "
            "d = Dims(64, 207, 12, 12, 1, 1, 1, 64, 20, 64, 3, 1); print(lib.mcrn_model_workspace_bytes(C.byref(d)))" % ROOT)
    sizes = {}
    for v in ("1", "0"):
        e = dict(os.environ)
        e["MCRN_FLAT_SETS"] = v
        sizes[v] = int(subprocess.run([sys.executable, "-c", code], env=e, capture_output=True, text=True, check=True).stdout.split()[-1])
    assert sizes["0"] < sizes["1"] - (1 << 30), sizes          # 21 pairs of plane sets less at METR-LA: > 1 GB


def test_launch_histogram_abi():
    from megacrn_amd import _lib
    _lib.launch_histogram(reset=True)
    assert _lib.launch_histogram() == {}          # (no GPU here: nothing launched since the reset)


def test_workspace_sizing_and_validation():
    from megacrn_amd._lib import lib, Dims
    d = Dims(64, 207, 12, 12, 1, 1, 1, 64, 20, 64, 3, 0)
    nb = lib.mcrn_model_workspace_bytes(C.byref(d))
    assert 1 << 28 < nb < 1 << 33          # ~1.5 GB of saved activations at METR-LA B=64
    d4 = Dims(64, 207, 12, 12, 1, 1, 1, 64, 20, 64, 4, 0)   # cheb_k = 4: two more planes per support than cheb_k = 3
    assert lib.mcrn_model_workspace_bytes(C.byref(d4)) > nb
    for bad in (1, 9):                                        # cheb_k = 1 is broken in the reference too; 2 .. 8 supported
        d2 = Dims(64, 207, 12, 12, 1, 1, 1, 64, 20, 64, bad, 0)
        assert lib.mcrn_model_workspace_bytes(C.byref(d2)) == 0
        assert b"cheb_k" in lib.mcrn_last_error()
    d3 = Dims(64, 207, 12, 12, 1, 1, 1, 64, 20, 64, 4, 2)    # the bf16 mode builds [S, 2SS - I]: cheb_k 2 or 3 only
    assert lib.mcrn_model_workspace_bytes(C.byref(d3)) == 0 and b"bf16" in lib.mcrn_last_error()
    assert lib.mcrn_cell_workspace_bytes(3, 13, 2, 8, 3) > 0
    assert lib.mcrn_agcn_workspace_bytes(3, 13, 9, 16, 1) == 0


def test_state_dict_layout_and_init_order_match_reference():
    """Same keys/shapes, and the same torch RNG consumption order as the reference constructor:
    with the golden's seed the non-bias parameters are bit-identical to the reference's."""
    import megacrn_amd
    rec, P, m = load_case("tiny", "f32")
    torch.manual_seed(1)   # seed used by tests/golden/make_golden.py for `tiny`
    model = megacrn_amd.MegaCRN(num_nodes=m["N"], input_dim=1, output_dim=1, horizon=m["T_out"],
                                rnn_units=m["H"], mem_num=m["M"], mem_dim=m["D"])
    sd = model.state_dict()
    assert list(sd.keys()) == list(P.keys())
    for k, v in sd.items():
        assert tuple(v.shape) == P[k].shape, k
        if not k.endswith("bias"):
            assert np.array_equal(v.numpy(), P[k]), k


def test_curriculum_draws_match_reference_stream():
    import megacrn_amd
    rec, P, m = load_case("odd", "f32")
    model = megacrn_amd.MegaCRN(num_nodes=m["N"], input_dim=1, output_dim=1, horizon=m["T_out"], rnn_units=m["H"],
                                mem_num=m["M"], mem_dim=m["D"], cl_decay_steps=m["cl_decay"]).train()
    np.random.seed(2 + 7)
    flags = model._teacher_flags(None, int(rec["batches_seen"]))
    assert [int(f) for f in flags] == rec["teacher"].tolist()
    model.eval()
    assert model._teacher_flags(None, 0) == [False] * m["T_out"]


def test_cpu_tensors_fail_loudly():
    import megacrn_amd
    model = megacrn_amd.MegaCRN(5, 1, 1, 2, 4)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        model(torch.randn(1, 2, 5, 1), torch.randn(1, 2, 5, 1))


def test_loader_shuffles_once_and_pads_with_last_sample():
    """model/utils.py:6-43 semantics of the counterpart DataLoader."""
    from megacrn_amd.train import DataLoader, StandardScaler
    xs = np.arange(10, dtype=np.float64).reshape(10, 1)
    ys = xs * 10
    dl = DataLoader(xs, ys, batch_size=4, shuffle=False)
    batches = list(dl.get_iterator())
    assert dl.size == 12 and dl.num_batch == 3
    assert batches[-1][0].ravel().tolist() == [8, 9, 9, 9]          # padded by repeating the last sample
    np.random.seed(0)
    dl = DataLoader(xs, ys, batch_size=4, shuffle=True)
    e1 = np.concatenate([b[0] for b in dl.get_iterator()]).ravel()
    e2 = np.concatenate([b[0] for b in dl.get_iterator()]).ravel()
    assert (e1 == e2).all() and sorted(e1.tolist()) == sorted([0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 9, 9])  # one permutation, reused
    assert (np.concatenate([b[1] for b in dl.get_iterator()]).ravel() == e1 * 10).all()
    sc = StandardScaler(mean=54.4, std=19.5)
    z = sc.transform(np.array([0.0, 54.4, 73.9]))
    np.testing.assert_allclose(sc.inverse_transform(z), [0.0, 54.4, 73.9], atol=1e-12)


def test_train_cli_defaults_match_reference_flags():
    from megacrn_amd.train import build_parser, synthetic_windows
    a = build_parser().parse_args([])
    assert (a.num_nodes, a.seq_len, a.horizon, a.rnn_units, a.mem_num, a.mem_dim) == (207, 12, 12, 64, 20, 64)
    assert (a.max_diffusion_step, a.batch_size, a.lr, a.epsilon, a.max_grad_norm) == (3, 64, 0.01, 1e-3, 5)
    assert a.steps == [50, 100] and a.lr_decay_ratio == 0.1 and a.patience == 20 and a.epochs == 200
    assert a.lamb == 0.01 and a.lamb1 == 0.01 and a.cl_decay_steps == 2000 and a.use_curriculum_learning is True
    x, y = synthetic_windows(5, 12, 7, 0)
    assert x.shape == (5, 12, 7, 2) and y.shape == (5, 12, 7, 2)
    assert (x[..., 0] == 0).mean() > 0.02 and 0 <= x[..., 1].min() and x[..., 1].max() < 1


def test_unchanged_reference_import_resolves_the_shim():
    """model/traintest_MegaCRN.py:15 is `from MegaCRN import MegaCRN` with the model directory on sys.path.
    With megacrn_amd/ first on sys.path instead, the same statement must yield the HIP-backed class,
    constructed with the trainer's get_model() keywords (:28-30).  Fresh interpreter, cwd outside the repo."""
    import subprocess
    import sys
    code = (
        "import sys; sys.path.insert(0, %r)\n"
        "from MegaCRN import MegaCRN\n"
        "import megacrn_amd.modules as mm\n"
        "assert MegaCRN is mm.MegaCRN\n"
        "m = MegaCRN(num_nodes=7, input_dim=1, output_dim=1, horizon=3, rnn_units=4, num_layers=1, mem_num=3,\n"
        "            mem_dim=4, cheb_k=3, cl_decay_steps=2000, use_curriculum_learning=True)\n"
        "assert list(m.state_dict())[:4] == ['memory.Memory', 'memory.Wq', 'memory.We1', 'memory.We2']\n"
        "import MegaCRN as shim\n"
        "assert all(hasattr(shim, n) for n in ('AGCN', 'AGCRNCell', 'ADCRNN_Encoder', 'ADCRNN_Decoder', 'print_params'))\n"
        "print('ok')\n") % os.path.join(ROOT, "megacrn_amd")
    r = subprocess.run([sys.executable, "-c", code], cwd="/tmp", capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stderr[-2000:]
    # and as a sub-module of the package (which rebinds the package attribute to the module: it stays constructible)
    code2 = ("import sys; sys.path.insert(0, %r)\n"
             "import megacrn_amd, megacrn_amd.modules as mm\n"
             "import megacrn_amd.MegaCRN as sub\n"
             "assert sub.MegaCRN is mm.MegaCRN\n"
             "m = megacrn_amd.MegaCRN(5, 1, 1, 2, 4)\n"
             "assert isinstance(m, mm.MegaCRN)\n"
             "print('ok')\n") % ROOT
    r = subprocess.run([sys.executable, "-c", code2], cwd="/tmp", capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stderr[-2000:]


def test_loader_scaler_and_prepare_match_reference_fixtures(golden_dir):
    """Counterpart DataLoader / StandardScaler / prepare_x_y host half against outputs of the reference's own
    model/utils.py:6-54 and traintest_MegaCRN.py:33-48 (tests/golden/make_golden_utils.py)."""
    from megacrn_amd.train import DataLoader, StandardScaler, split_x_y, build_parser
    z = np.load(f"{golden_dir}/utils_f32.npz")
    xs, ys = z["loader:xs"], z["loader:ys"]
    size, nbatch, bs, seed = [int(v) for v in z["loader:meta"]]
    np.random.seed(seed)
    dl = DataLoader(xs, ys, bs, shuffle=True)
    assert (dl.size, dl.num_batch) == (size, nbatch)
    assert np.array_equal(np.concatenate([b[0] for b in dl.get_iterator()]), z["loader:shuffled_x"])
    assert np.array_equal(np.concatenate([b[1] for b in dl.get_iterator()]), z["loader:shuffled_y"])
    assert np.array_equal(list(DataLoader(xs, ys, bs).get_iterator())[-1][0], z["loader:plain_x_last"])
    sc = StandardScaler(mean=xs[..., 0].mean(), std=xs[..., 0].std())
    assert np.array_equal(np.array([sc.mean, sc.std]), z["scaler:mean_std"])
    assert np.array_equal(sc.transform(xs[..., 0]), z["scaler:x0"])
    assert np.array_equal(sc.inverse_transform(sc.transform(xs[..., 0])), z["scaler:roundtrip"])
    args = build_parser().parse_args([])
    x0, y0, y1 = split_x_y(z["prep:x"], z["prep:y"], args)
    for got, want in ((x0, "prep:x0"), (y0, "prep:y0"), (y1, "prep:y1")):
        assert got.dtype == np.float32 and np.array_equal(got, z[want]), want
    # a rank's shard is the same slice of the same arrays
    x0s, y0s, y1s = split_x_y(z["prep:x"], z["prep:y"], args, 1, 3)
    assert np.array_equal(x0s, z["prep:x0"][1:3]) and np.array_equal(y1s, z["prep:y1"][1:3])


def test_trainer_rejects_malformed_inputs_before_touching_the_library():
    """FlatTrainer / MegaCRN.forward hand raw pointers to the C ABI: wrong shapes, dtypes and devices must raise
    like the reference's torch.cat / stack would, not read out of bounds."""
    import megacrn_amd
    m = megacrn_amd.MegaCRN(5, 1, 1, 3, 4)
    x, yc, y = torch.randn(2, 4, 5, 1), torch.randn(2, 3, 5, 1), torch.randn(2, 3, 5, 1)
    for bad in ((x, yc[:, :2], y), (x, torch.randn(2, 3, 5, 2), y), (x, yc, torch.randn(3, 3, 5, 1)),
                (torch.randn(2, 4, 6, 1), yc, y)):
        with pytest.raises(ValueError):
            m._check_inputs(*bad)
    m._check_inputs(x, yc, y)
    m._check_inputs(x, yc, None)


def test_shipped_kernels_use_no_packed_fp32_valu():
    """Build guard (csrc/Makefile: -fno-slp-vectorize -fno-vectorize): the library is built without packed-fp32 VALU instructions.
    Since round 5 this is a measured PERFORMANCE choice - the same library with the vectorisers on ran 0.5 - 1.1 % slower on METR-LA,
    PEMS-BAY and EXPY-TKY in one call (profiles/r5/experiments.md section 1): a packed-fp32 op beside MFMAs costs +22 .. 26 cycles,
    MI355X_MICROARCH.md - not a correctness one: round 2's wrong high halves beside a foreign MFMA stream did not reproduce in
    rounds 4 and 5 and that finding is retired.  A build that lost the flags would silently give the percent back: checked here."""
    import re
    import shutil
    import subprocess
    import tempfile
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    so = os.path.join(root, "megacrn_amd", "libmegacrn_hip.so")
    objcopy, objdump = "/opt/rocm/lib/llvm/bin/llvm-objcopy", "/opt/rocm/lib/llvm/bin/llvm-objdump"
    if not (os.path.exists(so) and os.path.exists(objcopy) and os.path.exists(objdump)):
        pytest.skip("library or LLVM binutils not present")
    tmp = tempfile.mkdtemp()
    try:
        fat = os.path.join(tmp, "fatbin.bin")
        subprocess.run([objcopy, "--dump-section", f".hip_fatbin={fat}", so, os.path.join(tmp, "copy.so")], check=True)
        data = open(fat, "rb").read()
        starts = [m.start() for m in re.finditer(b"\x7fELF", data)]
        assert starts, "no device code objects found in the library"
        nmfma = 0
        for n, i in enumerate(starts):
            end = starts[n + 1] if n + 1 < len(starts) else len(data)
            img = os.path.join(tmp, f"co{n}.elf")
            open(img, "wb").write(data[i:end])
            dis = subprocess.run([objdump, "-d", img], capture_output=True, text=True, check=True).stdout
            bad = re.findall(r"v_pk_(?:mul|fma|add)_f32", dis)
            assert not bad, f"code object {n}: {len(bad)} packed-fp32 VALU instructions"
            nmfma += len(re.findall(r"v_mfma", dis))
        assert nmfma > 1000          # we really looked at the kernels
    finally:
        shutil.rmtree(tmp, ignore_errors=True)


def test_shipped_kernels_do_not_spill():
    """Build guard: no GEMM-shaped or streaming kernel of the shipped library uses scratch (register spills), and the few fused-propagation
    variants that do stay within what was measured.  Round 5 shipped, for a few commits, a 256x256 ping-pong bf16 GEMM tile with 556 B/lane
    of scratch after an accumulator-preload edit: every parity test passed and the bf16-mode step was simply a tenth slower
    (profiles/r5/experiments.md section 10).  tools/scratch_report.py reads the sizes from the code objects' metadata."""
    import importlib.util
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    so = os.path.join(root, "megacrn_amd", "libmegacrn_hip.so")
    spec = importlib.util.spec_from_file_location("scratch_report", os.path.join(root, "tools", "scratch_report.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    if not (os.path.exists(so) and os.path.exists(mod.READELF)):
        pytest.skip("library or LLVM binutils not present")
    sizes = mod.scratch_sizes(so)
    assert len(sizes) > 200 and any(k.startswith("gemm_bf16_pp_kernel<") for k in sizes)      # we really looked at the kernels
    # known, measured spills of the widest fused two-hop variants (K = 3 planes of a 7- or 8-fragment adjacency row band) and one d-grad form
    # (round 6: the bodies of the fused two-hop kernels as device functions and the d-grad's output forms as a template parameter removed the
    #  other three; what is left is the widest propagation variant and the hoisted-backward form of the widest d-grad)
    allowed = {"prop2_fwd_kernel<8, 3>": 8, "dgrad_stream_kernel<8, 2, 2>": 12}
    bad = {k: v for k, v in sizes.items() if v > allowed.get(k, 0)}
    assert not bad, f"kernels with new register spills (bytes per lane): {bad}"


def test_shipped_kernels_have_no_valu_sgpr_to_vmem_hazard():
    """Build guard for the inline-asm loads (prop_small.h's streamed adjacency fragments, the LDS-DMA issue blocks): a VMEM
    instruction that reads an SGPR pair written by a VALU instruction (v_readfirstlane / v_readlane ...) needs 5 wait states,
    and the compiler's hazard recogniser cannot see into asm text.  Round 4 found the forward propagation of 256 < N <= 352
    and several new variants one k-step wrong from exactly this (tools/isa_hazards.py; tools/kbench/prop1_test)."""
    import importlib.util
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    so = os.path.join(root, "megacrn_amd", "libmegacrn_hip.so")
    spec = importlib.util.spec_from_file_location("isa_hazards", os.path.join(root, "tools", "isa_hazards.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    if not (os.path.exists(so) and os.path.exists(mod.OBJCOPY) and os.path.exists(mod.OBJDUMP)):
        pytest.skip("library or LLVM binutils not present")
    # the scanner itself: a planted hazard is found, the same sequence behind s_nop 4 is not
    planted = ("0000 <k>:\n\tv_readfirstlane_b32 s2, v66    // 0\n\tv_readfirstlane_b32 s3, v67    // 4\n"
               "\tglobal_load_dwordx4 v[66:69], v126, s[2:3]    // 8\n")
    assert len(mod.scan_disassembly(planted)) == 1
    assert not mod.scan_disassembly(planted.replace("\tglobal_load", "\ts_nop 4    // 6\n\tglobal_load"))
    hits, nloads = mod.scan_library(so)
    assert nloads > 1000                      # we really looked at the kernels
    assert not hits, f"{len(hits)} VALU-SGPR -> VMEM hazards, first: {hits[0]}"


def _device_code_objects(tmp):
    """(path, disassembler) of every gfx950 code object inside the shipped library, or None when tools are absent."""
    import re
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    so = os.path.join(root, "megacrn_amd", "libmegacrn_hip.so")
    objcopy = "/opt/rocm/lib/llvm/bin/llvm-objcopy"
    if not (os.path.exists(so) and os.path.exists(objcopy)):
        return None
    fat = os.path.join(tmp, "fatbin.bin")
    subprocess.run([objcopy, "--dump-section", f".hip_fatbin={fat}", so, os.path.join(tmp, "copy.so")], check=True)
    data = open(fat, "rb").read()
    starts = [m.start() for m in re.finditer(b"\x7fELF", data)]
    out = []
    for n, i in enumerate(starts):
        end = starts[n + 1] if n + 1 < len(starts) else len(data)
        img = os.path.join(tmp, f"co{n}.elf")
        open(img, "wb").write(data[i:end])
        out.append(img)
    return out


def _vregs(operand_text):
    """Set of VGPR numbers named in an operand string (v7, v[10:13])."""
    import re
    regs = set()
    for a, b in re.findall(r"\bv\[(\d+):(\d+)\]", operand_text):
        regs.update(range(int(a), int(b) + 1))
    regs.update(int(a) for a in re.findall(r"\bv(\d+)\b", operand_text))
    return regs


def check_register_ring_contract(asm_lines):
    """The WIDE fused propagation (prop_small.h: 256 < N <= 352) streams its adjacency fragments with inline-asm
    `global_load_dwordx4 vDST, vOFF, s[base]` into a register ring and waits with hand-counted `s_waitcnt vmcnt(n)` in
    separate asm statements.  That is only correct if (1) no instruction touches a ring destination while its load
    is still outstanding - a register copy or spill in between would read data that has not landed - and (2) the counted
    waits see exactly the VMEM operations the source assumes.  Replays the wave's vmcnt queue over the straight-line
    instruction stream: every VMEM instruction enters the FIFO, `s_waitcnt vmcnt(n)` retires all but the youngest n.
    Returns (number of ring loads checked, list of violations)."""
    import re
    fifo = []                      # outstanding VMEM ops, oldest first: set of destination VGPRs (empty for stores)
    ring, bad = 0, []
    for ln in asm_lines:
        m = re.match(r"\s+(\S+)\s*(.*?)\s*//", ln)
        if not m:
            continue
        op, args = m.group(1), m.group(2)
        if op == "s_waitcnt":
            c = re.search(r"vmcnt\((\d+)\)", args)
            if c:
                keep = int(c.group(1))
                fifo = fifo[len(fifo) - keep:] if keep < len(fifo) else fifo
            continue
        touched = _vregs(args)
        for dst in fifo:
            if dst and dst & touched:
                bad.append(ln.strip()[:90])
                break
        if re.match(r"(global|buffer|flat|scratch)_(load|store|atomic)", op):
            is_ring = op == "global_load_dwordx4" and re.search(r",\s*v\d+,\s*s\[\d+:\d+\]", args) is not None
            dst = _vregs(args.split(",")[0]) if "_load" in op else set()
            fifo.append(dst if is_ring else set())
            ring += is_ring
    return ring, bad


def test_register_ring_checker_catches_an_early_read():
    ok = ["\tglobal_load_dwordx4 v[4:7], v1, s[2:3]    // 0", "\tv_add_u32 v9, v8, v8    // 0", "\ts_waitcnt vmcnt(0)    // 0",
          "\tv_mov_b32 v10, v4    // 0"]
    assert check_register_ring_contract(ok) == (1, [])
    early = [ok[0], "\tv_mov_b32 v10, v4    // 0", ok[2]]
    assert len(check_register_ring_contract(early)[1]) == 1
    counted = [ok[0], "\tglobal_load_dwordx4 v[12:15], v1, s[2:3] offset:1024    // 0", "\ts_waitcnt vmcnt(1)    // 0",
               "\tv_mov_b32 v10, v5    // 0", "\tv_mov_b32 v11, v13    // 0"]
    assert len(check_register_ring_contract(counted)[1]) == 1          # v13 belongs to the load still in flight


def test_wide_fused_propagation_register_ring_contract():
    """ADVICE (round 2): make the inline-asm register ring of prop2_{fwd,bwd}_kernel<9..11, 2> checkable on every build:
    no scratch / VGPR spills in those kernels, and no instruction touches a ring register between its load and the
    counted wait that retires it."""
    import re
    import shutil
    import subprocess
    import tempfile
    objdump, readelf = "/opt/rocm/lib/llvm/bin/llvm-objdump", "/opt/rocm/lib/llvm/bin/llvm-readelf"
    tmp = tempfile.mkdtemp()
    try:
        cos = _device_code_objects(tmp)
        if not cos or not (os.path.exists(objdump) and os.path.exists(readelf)):
            pytest.skip("library or LLVM binutils not present")
        want = [f"_ZN4mcrn16prop2_{d}_kernelILi{nf}ELi2EEEvNS_6Prop2PE" for d in ("fwd", "bwd") for nf in (9, 10, 11)]
        seen = 0
        for img in cos:
            notes = subprocess.run([readelf, "--notes", img], capture_output=True, text=True, check=True).stdout
            for sym in want:
                if sym not in notes:
                    continue
                seen += 1
                meta = notes[:notes.index(sym)]
                meta = meta[meta.rindex("- .agpr_count") if "- .agpr_count" in meta else 0:] + notes[notes.index(sym):notes.index(sym) + 600]
                priv = re.search(r"\.private_segment_fixed_size:\s+(\d+)", meta)
                vsp = re.search(r"\.vgpr_spill_count:\s+(\d+)", meta)
                assert priv and int(priv.group(1)) == 0, (sym, "scratch in a register-ring kernel")
                assert vsp is None or int(vsp.group(1)) == 0, (sym, "VGPR spills in a register-ring kernel")
                dis = subprocess.run([objdump, "-d", f"--disassemble-symbols={sym}", img], capture_output=True, text=True,
                                     check=True).stdout.splitlines()
                ring, bad = check_register_ring_contract(dis)
                assert ring >= 20, (sym, ring)             # 2 loads per k-step, >= 18 k-steps per hop
                assert not bad, (sym, bad[:5])
        assert seen == len(want), f"only {seen} of {len(want)} wide propagation kernels found in the library"
    finally:
        shutil.rmtree(tmp, ignore_errors=True)
