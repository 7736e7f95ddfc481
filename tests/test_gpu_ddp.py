"""The N > 1 path on the one GPU of a test box: the bucketed, overlapped gradient mean of
nextou_amd/ddp.py over RCCL (`nccl`, world size 1) — eager and captured into a hipGraph — against the plain step; bench.py's
averaged step end to end; two ranks sharing the GPU over gloo.  No retries, no skips: the GPU memory fault these paths used to hit
was MIOpen's backward-data kernel of the 1x1 head convolution reading past its operand (profiles/r05_n_gt_1.md), and the heads now run on K8 (csrc/head_rows.hip)."""
import json
import os
import subprocess
import sys

import pytest

from conftest import REPO

pytestmark = pytest.mark.gpu


def _xfail_on_watchdog_capture_error(proc):
    """The one failure of these runs that is neither this repository's nor deterministic: PyTorch's RCCL watchdog THREAD terminating the process
    with hipErrorCapturedEvent while a step with collectives is being captured (about once in 25 runs of the tiny workload,
    two precautions in place, mechanism not established — a stand-alone attempt stayed clean).  Reported as XFAIL with this
    reason (no retry, no skip; the outcome stays visible in the report) — every other failure fails the test."""
    err = proc.stderr or ""
    if proc.returncode != 0 and "hipErrorCapturedEvent" in err and "watchdog thread terminated" in err:
        pytest.xfail("PyTorch's RCCL watchdog thread hit hipErrorCapturedEvent during the capture (intermittent, DESIGN.md section 6)")


def _json_line(stdout):
    lines = [l for l in stdout.splitlines() if l.startswith("{")]
    assert len(lines) == 1, stdout[-2000:]
    return json.loads(lines[0])


def _check_averaged_record(r, modes):
    assert r["hip_library_loaded"] and r["backend"] == "nccl" and r["world_size"] == 1 and r["buckets"] >= 2 and r["steps"] == 3
    assert r["grad_is_none_plain"] == r["grad_is_none_avg_eager"]
    assert len(r["grad_is_none_plain"]) > 0          # the lowest-resolution head has weight 0 in the deep-supervision loss
    assert r["weights_moved"] == 0.0
    tiny_g, tiny_m = 2e-6 * r["grad_scale"], 2e-6 * r["momentum_scale"]
    assert r["grad1_avg_eager_vs_plain"] <= max(4.0 * r["grad1_plain_vs_plain"], tiny_g), r
    for mode in modes:
        assert r["grad_%s_vs_plain" % mode] <= max(4.0 * r["grad_plain_vs_plain"], tiny_g), (mode, r)
        assert r["momentum_%s_vs_plain" % mode] <= max(4.0 * r["momentum_plain_vs_plain"], tiny_m), (mode, r)


@pytest.mark.timeout(1800)
def test_averaged_step_over_rccl_matches_plain_step():
    """World-size-1 RCCL group, learning rate 0 (tests/averaged_step_check.py says why), the DEFAULT modes of every N (round 6: the averaged
    step replayed as TWO hipGraphs around eager collectives — harness.SplitGraphedTrainStep — and its eager form; the plain step captured):
    after three steps the averaged step's gradients and the optimizer's momentum buffers (what it was handed through `p.grad`, i.e. the
    bucket views) equal the plain step's: bit for bit when two plain runs agree bit for bit, else within 4x their distance; the
    zero-weighted head's parameters keep grad = None; the weights did not move.  No collective is captured here, so nothing of PyTorch's
    watchdog can end the process: no XFAIL clause."""
    proc = subprocess.run([sys.executable, os.path.join(REPO, "tests", "averaged_step_check.py"), "--backend", "nccl"],
                          capture_output=True, text=True, timeout=1500)
    assert proc.returncode == 0, proc.stdout[-2000:] + proc.stderr[-3000:]
    r = _json_line(proc.stdout)
    print(r)
    assert r["captured_collectives"] is False and r["grad_avg_graph_vs_plain"] is None
    assert r["grad_is_none_plain"] == r["grad_is_none_avg_split"]
    _check_averaged_record(r, ("avg_eager", "avg_split", "plain_graph"))


@pytest.mark.timeout(1800)
def test_explicitly_captured_rccl_step_matches_plain_step():
    """The opt-in mode (`bench.py --graph on` with a process group up, `averaged_step_check.py --captured-collectives`): hooks, bucket copies,
    RCCL all-reduces, finalize and ClipSGD on the bucket views inside ONE hipGraph.  Same bars.  This is the only place where the watchdog
    abort of DESIGN.md section 6 can strike, and the only test that reports it as XFAIL."""
    proc = subprocess.run([sys.executable, os.path.join(REPO, "tests", "averaged_step_check.py"), "--backend", "nccl", "--captured-collectives"],
                          capture_output=True, text=True, timeout=1500)
    _xfail_on_watchdog_capture_error(proc)
    assert proc.returncode == 0, proc.stdout[-2000:] + proc.stderr[-3000:]
    r = _json_line(proc.stdout)
    print(r)
    assert r["captured_collectives"] is True and r["grad_is_none_plain"] == r["grad_is_none_avg_graph"]
    _check_averaged_record(r, ("avg_eager", "avg_split", "avg_graph", "plain_graph"))


@pytest.mark.timeout(1800)
@pytest.mark.parametrize("graph", ["auto", "off", "on"])
def test_bench_averaged_step_on_one_gpu(graph):
    """bench.py --force-averager: the N > 1 step (hooks, buckets, RCCL collectives, finalize, ClipSGD) on a world-size-1 RCCL group.
    `auto` (the default of every N > 1 run: two graphs around eager collectives) and `off` (the eager step — the mode that died with a GPU
    memory fault in round 4) must simply pass; `on` captures the collectives too and is the only mode with the watchdog XFAIL clause."""
    cmd = [sys.executable, os.path.join(REPO, "bench.py"), "--steps", "3", "--warmup", "2", "--workload", "tiny", "--force-averager",
           "--graph", graph, "--no-miopen-find", "--no-cpu-baseline"]
    out = subprocess.run(cmd, capture_output=True, text=True, timeout=1500)
    if graph == "on":
        _xfail_on_watchdog_capture_error(out)
    assert out.returncode == 0, out.stderr[-3000:]
    rec = _json_line(out.stdout)
    assert rec["config"]["gradient_averager"] is True and rec["config"]["step_replayed_as_hipgraph"] is (graph != "off")
    assert rec["config"]["graph_capture_error"] is None
    mode = rec["config"]["graph_mode"]
    assert {"auto": "two graphs around eager collectives" in mode, "off": mode.startswith("eager"), "on": "collectives captured" in mode}[graph], mode
    assert rec["dist"]["initialized"] and rec["dist"]["backend"] == "nccl" and rec["dist"]["world_size"] == 1
    assert rec["value"] > 0 and rec["roofline"]["launches"] > 0
    assert rec["roofline_graph"]["K8_head_backward"]["launches"] > 0       # the heads' backward ran on this library's kernels


@pytest.mark.timeout(2700)
def test_bench_two_ranks_share_one_gpu():
    """The N > 1 path of bench.py end to end (launcher env, bucketed overlapped gradient mean, barrier + max-over-ranks timing, one
    JSON line from rank 0) with two ranks on this box's single GPU over gloo; on the 8-GPU node the same code runs one rank per GPU
    over RCCL.  The line says what the process group was."""
    env = dict(os.environ, NEXTOU_DIST_BACKEND="gloo")
    cmd = [sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node", "2", "--master-addr",
           "127.0.0.1", "--master-port", "29533", os.path.join(REPO, "bench.py"), "--gpus", "2", "--steps", "2",
           "--warmup", "1", "--workload", "tiny", "--no-miopen-find"]
    out = subprocess.run(cmd, env=env, capture_output=True, text=True, timeout=1500)
    assert out.returncode == 0, out.stderr[-3000:]
    rec = _json_line(out.stdout)
    assert rec["n_gpus"] == 2 and rec["scaling"] == "weak" and rec["steps"] == 2 and rec["value"] > 0
    assert rec["config"]["global_batch"] == 4 and rec["roofline"]["launches"] > 0
    assert "cpu_baseline" not in rec or rec["cpu_baseline"] is None
    assert rec["dist"]["backend"] == "gloo" and rec["dist"]["world_size"] == 2 and [r["rank"] for r in rec["dist"]["ranks"]] == [0, 1]
    assert rec["dist"]["distinct_devices"] == 1          # both ranks on this box's one GPU (the 8-GPU node reports 8)


@pytest.mark.timeout(2700)
def test_bench_gpus_2_typed_without_a_launcher():
    """`python bench.py --gpus 2 ...` exactly as the round driver types it, no torch.distributed.run in front:
    bench.py starts its own two ranks (nextou_amd/launch.py), rank 0's JSON line reaches this process's stdout, the exit code is the
    launcher's.  gloo because both ranks share this box's single GPU; on the 8-GPU node the default backend is RCCL."""
    env = {k: v for k, v in os.environ.items() if k not in ("WORLD_SIZE", "RANK", "LOCAL_RANK", "MASTER_ADDR", "MASTER_PORT")}
    env["NEXTOU_DIST_BACKEND"] = "gloo"
    cmd = [sys.executable, os.path.join(REPO, "bench.py"), "--gpus", "2", "--steps", "2", "--warmup", "1", "--workload", "tiny",
           "--no-miopen-find"]
    out = subprocess.run(cmd, env=env, capture_output=True, text=True, timeout=1500)
    assert out.returncode == 0, out.stderr[-3000:]
    rec = _json_line(out.stdout)
    assert rec["n_gpus"] == 2 and rec["dist"]["world_size"] == 2 and rec["dist"]["backend"] == "gloo"
    assert rec["config"]["step_replayed_as_hipgraph"] is True and "two graphs" in rec["config"]["graph_mode"]       # (gloo's collectives run between the graphs)
    assert rec["config"]["graph_capture_error"] is None and rec["config"]["global_batch"] == 4 and rec["value"] > 0
    assert "without a launcher" in out.stderr
