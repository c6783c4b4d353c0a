"""The 8-bit key / value cache where a user meets it: conversations, tensor-parallel ranks, and the command lines of the llm example."""
import json
import os
import re
import signal
import subprocess
import sys
import time
import urllib.request

import pytest
import torch

from test_kv8_engine import KINDS, gpu, model, tokens
from zml_b200 import ops
from zml_b200.serving import Engine
from zml_b200.serving.engine import Session

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MAIN, SERVE = (os.path.join(ROOT, "examples", "llm", n) for n in ("main.py", "serve.py"))


# ------------------------------------------------------------------ conversations
def check_session(kind, device):
    """Two turns: blocks of decode steps read the tokens that single steps do, and the second turn goes on over what the first one has cached."""
    m = model(device=device)
    got = []
    for interval in (1, 5):
        s = Session(Engine(m, num_pages=40, page_size=16, max_batch=1, max_seq_len=512, kv_dtype=kind), 400)
        for n in (70, 33):
            s.run_prefill(tokens(n, n))
            got.append(s.run_decode(max_new_tokens=9, stream_interval=interval))
        s.close()
    assert got[:2] == got[2:] and all(len(t) == 9 for t in got)


@KINDS
def test_conversations_cpu(kind):
    check_session(kind, "cpu")


@gpu
@KINDS
def test_conversations(kind):
    check_session(kind, "cuda")
    ops.raise_on_status()


# ------------------------------------------------------------------ tensor-parallel ranks
_TP_WORKER = r"""
import os, sys, torch
sys.path[:0] = [os.environ["ZB_ROOT"], os.path.join(os.environ["ZB_ROOT"], "tests")]
from test_kv8_engine import FAMILIES, off, tokens
from zml_b200.parallel.comm import Comm
from zml_b200.serving import Engine
c = Comm.from_env(backend="gloo")
single = Comm.single(torch.device("cpu"))
for family in ("llama", "qwen3_moe"):
    config, cls, preset = FAMILIES[family]
    for kind in ("fp8", "int8"):
        got = {}
        for label, comm in (("tp", c), ("single", single)):
            m = cls(config.from_hf(dict(preset)), comm, device="cpu", dtype=torch.bfloat16).init_random(seed=3, std=0.05)
            e = Engine(m, num_pages=32, page_size=16, max_batch=2, max_seq_len=128, kv_dtype=kind)
            k = e.kv_cache[0, 0].codes
            assert k.shape[1] == (m.config.num_key_value_heads if hasattr(m.config, "num_key_value_heads") else m.config.hkv) // comm.world, k.shape
            r, prompt = e.open_request(), tokens(60)
            got[label] = torch.stack([e.step([(r, prompt[a:b])], [[b - a - 1]])[0].float() for a, b in ((0, 40), (40, 41), (41, 59), (59, 60))])
        for a, b in zip(got["tp"], got["single"]):
            assert off(a, b) < 0.05, (family, kind, off(a, b))
        same = c.all_gather_object(got["tp"])
        assert all(torch.equal(s, same[0]) for s in same)
print("KV8_TP_OK", c.rank, flush=True)
c.finish(0)
"""


def test_two_ranks_hold_their_heads_of_the_cache(tmp_path):
    """Each of two gloo ranks has a cache of its own key heads; logits of prompts, portions and single tokens are those of one rank with all heads.  Rows are
    scaled one by one, so a rank's rows are the whole model's; what differs are sums over ranks that are rounded to bf16 (2^-8 an activation, through
    two layers), and codes that such a rounding moves by a step."""
    script = tmp_path / "w.py"
    script.write_text(_TP_WORKER)
    r = subprocess.run([sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node=2", "--master-addr", "127.0.0.1", "--master-port", "29677",
                        str(script)], capture_output=True, text=True, env=dict(os.environ, ZB_ROOT=ROOT), timeout=300)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-3000:]
    assert r.stdout.count("KV8_TP_OK") == 2


# ------------------------------------------------------------------ command lines
def repo(path):
    from test_llm_cli import make_repo
    make_repo(str(path))
    return f"--model={path}"


def prompt(args):
    return subprocess.run([sys.executable, MAIN, "--prompt=hello world the quick brown fox", "--seqlen=256", "--max-new-tokens=6", *args], capture_output=True,
                          text=True, timeout=300)


def test_command_lines_refuse_what_takes_no_such_cache(tmp_path):
    """On the CPU models are fp32; other backends read the bf16 cache; other types are unknown.  Each says so and ends."""
    pytest.importorskip("tokenizers")
    at = repo(tmp_path)
    for args, words in ((["--cpu", "--kv-cache=fp8"], "bfloat16"), (["--cpu", "--kv-cache=fp8", "--backend=vanilla"], "b200 backend")):
        r = prompt([at, *args])
        assert r.returncode != 0 and words in r.stderr, r.stderr[-2000:]
    r = subprocess.run([sys.executable, SERVE, at, "--cpu", "--port=0", "--kv-cache=int8"], capture_output=True, text=True, timeout=300)
    assert r.returncode != 0 and "bfloat16" in r.stderr, r.stderr[-2000:]


@gpu
def test_command_lines(tmp_path):
    pytest.importorskip("tokenizers")
    at = repo(tmp_path)
    for kind in ("fp8", "int8"):
        r = prompt([at, f"--kv-cache={kind}"])
        assert r.returncode == 0 and "tok/s" in r.stdout, r.stderr[-2000:]
    r = prompt([at, "--kv-cache=e5m2"])
    assert r.returncode != 0 and "unknown cache type" in r.stderr, r.stderr[-2000:]
    p = subprocess.Popen([sys.executable, SERVE, at, "--port=0", "--max-batch=2", "--seqlen=256", "--kv-cache=int8"], stderr=subprocess.PIPE,
                         stdout=subprocess.PIPE, text=True)
    try:
        port, t0 = None, time.time()
        while port is None and time.time() - t0 < 120:
            line = p.stderr.readline()
            if not line and p.poll() is not None:
                break
            found = re.search(r"http://127\.0\.0\.1:(\d+)", line)
            port = int(found.group(1)) if found else None
        assert port, "the server did not come up"
        ask = urllib.request.Request(f"http://127.0.0.1:{port}/v1/completions", data=json.dumps({"prompt": "hello world", "max_tokens": 5}).encode())
        with urllib.request.urlopen(ask, timeout=120) as r:
            assert json.loads(r.read())["usage"]["completion_tokens"] == 5
        p.send_signal(signal.SIGTERM)
        assert p.wait(timeout=60) == 0
    finally:
        if p.poll() is None:
            p.kill()
