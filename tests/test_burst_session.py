"""infer_burst --model session: the cache's operators as a client calls
them, on the CPU and, with -m gpu, on an MI355X."""

from __future__ import annotations

import json
import shutil
import subprocess
import sys

import pytest
import torch

from nvshare_amd.paths import REPO_ROOT, artifacts, ensure_kernels
from nvshare_amd.workloads import infer_burst
from nvshare_amd.workloads.session import Sessions


@pytest.fixture(scope="module", autouse=True)
def kernels():
    ensure_kernels()


def run(*args):
    r = subprocess.run(
        [sys.executable, "-m", "nvshare_amd.workloads.infer_burst",
         "--model", "session", "--think-s", "0.05", *args],
        capture_output=True, text=True, timeout=240)
    assert r.returncode == 0, r.stderr[-3000:]
    assert "PASS" in r.stdout
    return json.loads(r.stdout.strip().splitlines()[-1])


def test_session_cpu():
    res = run("--device", "cpu", "--batch", "2", "--bursts", "2",
              "--infers-per-burst", "3", "--prompt", "9", "--layers", "2",
              "--heads", "4", "--kv-heads", "2", "--head-dim", "64",
              "--page", "16")
    assert res["infers"] == 8 and res["tokens"] == 2 * 2 * 12


ALONE = """
import pathlib, sys
from nvshare_amd import paths
paths.HIP_BUILD_DIR = pathlib.Path(sys.argv[1])
"""


def alone(tmp_path, code, *args):
    """Runs the code where the kernels' library has not been built."""
    shutil.copy(artifacts().kvbind, tmp_path)
    return subprocess.run(
        [sys.executable, "-c", ALONE + code, str(tmp_path), *args],
        capture_output=True, text=True, timeout=240, cwd=REPO_ROOT)


def test_session_cpu_without_kernels(tmp_path):
    r = alone(tmp_path, """
from nvshare_amd.workloads.infer_burst import main
main(sys.argv[2:])
""", "--model", "session", "--device", "cpu", "--batch", "1", "--bursts",
              "1", "--infers-per-burst", "1", "--prompt", "3", "--layers",
              "1", "--heads", "1", "--kv-heads", "1", "--head-dim", "64",
              "--think-s", "0")
    assert r.returncode == 0, r.stderr[-3000:]


@pytest.mark.gpu
def test_launch_without_kernels_is_an_error(tmp_path):
    r = alone(tmp_path, """
import torch
from nvshare_amd import kvcache
cache = kvcache.PagedCache.empty(2, 16, 1, 64)
q = torch.zeros(1, 1, 64, dtype=torch.bfloat16, device="cuda")
one = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
for call in (lambda: kvcache.attend(cache, q, one, one[0]),
             lambda: kvcache.append(cache, q, q, one, one[0])):
    try:
        call()
    except RuntimeError as e:
        assert "libnvshare_hiputil.so" in str(e), e
        assert "make -C hip" in str(e), e
    else:
        raise SystemExit("no error")
""")
    assert r.returncode == 0, r.stderr[-3000:]


@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_session_notices_a_changed_cache(cache):
    m = Sessions(2, 40, layers=1, heads=2, kv_heads=1, dim=64, page=16,
                 cache=cache, device="cpu")
    m.step(19)
    before = m.fingerprint()
    m.check()
    page = int(m.table[1, 1])
    m.caches[0].v.view(torch.uint8)[page, 5] ^= 1  # behind the last token
    assert m.fingerprint() == before
    m.caches[0].v.view(torch.uint8)[page, 2] ^= 1
    assert m.fingerprint() != before


@pytest.mark.parametrize("cache", ["same", "e4m3"])
def test_session_notices_exchanged_places(cache):
    """Pages of two sessions, pages of one, rows, and words exchanged."""
    m = Sessions(2, 40, layers=1, heads=2, kv_heads=1, dim=64, page=16,
                 cache=cache, device="cpu")
    m.step(35)
    before = m.fingerprint()
    k = m.caches[0].k.view(torch.uint8)
    (a, b), c = m.table[:, 0].tolist(), int(m.table[0, 1])
    for one, other in (((a,), (b,)), ((a,), (c,)), ((a, 3), (a, 9)),
                       ((a, 3, 0, slice(0, 4)), (a, 3, 0, slice(8, 12)))):
        held = k.clone()
        k[one], k[other] = held[other], held[one]
        assert m.fingerprint() != before
        k.copy_(held)
        assert m.fingerprint() == before
    m.caches[0] = m.caches[0]._replace(k=m.caches[0].v, v=m.caches[0].k)
    assert m.fingerprint() != before


def test_session_notices_a_wrong_answer():
    m = Sessions(1, 40, layers=1, heads=2, kv_heads=1, dim=64, page=16,
                 device="cpu")
    m.step(30)
    m.answer[2][3, 1, 7] += 0.5
    with pytest.raises(SystemExit):
        m.check()


def test_other_models_stay(capsys):
    infer_burst.main(["--device", "cpu", "--model", "tiny", "--batch", "1",
                      "--image", "32", "--bursts", "1",
                      "--infers-per-burst", "1", "--think-s", "0"])
    assert json.loads(capsys.readouterr().out.splitlines()[-1])[
        "infers"] == 1


@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["same", "e4m3"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_session_gpu(cache, dtype):
    if not torch.cuda.is_available():
        pytest.skip("no GPU here")
    res = run("--batch", "4", "--bursts", "2", "--infers-per-burst", "10",
              "--prompt", "300", "--cache", cache, "--dtype", dtype)
    assert res["infers"] == 22 and res["tokens"] == 4 * 2 * 310


@pytest.mark.parametrize("name", ["batch", "bursts", "prompt", "layers",
                                  "page"])
def test_session_refuses_sizes_below_one(name, capsys):
    with pytest.raises(SystemExit):
        infer_burst.main(["--model", "session", "--device", "cpu",
                          f"--{name}", "0"])
    assert f"--{name} 0" in capsys.readouterr().err


@pytest.mark.parametrize("args,said", [
    (("--infers-per-burst", "-3"), "--infers-per-burst -3"),
    (("--heads", "0"), "--heads 0"),
    (("--kv-heads", "0"), "--kv-heads 0"),
    (("--heads", "6", "--kv-heads", "4"), "no multiple of --kv-heads 4"),
    (("--head-dim", "80"), "--head-dim 80"),
    (("--think-s", "-1"), "--think-s -1"),
])
def test_session_refuses_what_it_cannot_run(args, said, capsys):
    """A turn of a prompt less some tokens had pages for those only."""
    with pytest.raises(SystemExit):
        infer_burst.main(["--model", "session", "--device", "cpu",
                          "--prompt", "4", "--bursts", "2", "--layers", "1",
                          "--batch", "1", *args])
    assert said in capsys.readouterr().err


def test_session_without_single_tokens(capsys):
    infer_burst.main(["--model", "session", "--device", "cpu", "--batch",
                      "1", "--bursts", "2", "--infers-per-burst", "0",
                      "--prompt", "5", "--layers", "1", "--heads", "2",
                      "--kv-heads", "2", "--head-dim", "64", "--think-s",
                      "0"])
    assert json.loads(capsys.readouterr().out.splitlines()[-1])[
        "tokens"] == 10
