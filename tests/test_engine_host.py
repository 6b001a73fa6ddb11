"""Host code of engines and operators on a CUDA runtime of host memory (fake_cudart.c, preloaded
into a child process): what they do when a call fails, without a GPU."""
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
PRELUDE = """
import ctypes, sys, types
sys.path.insert(0, {pkg!r})
class Array:  # what Engine needs of a torch tensor
    def __init__(self, a): self.a = a
    def to(self, where): return self
    def data_ptr(self): return self.a.ctypes.data
sys.modules['torch'] = types.SimpleNamespace(from_numpy=Array)
from ijb200 import lib, synth
from ijb200.engine import Engine
F = ctypes.CDLL({fake!r})
F.fake_call.restype = ctypes.c_char_p
F.fake_value.restype = ctypes.c_size_t
def log(start=0):
    return [(F.fake_call(i).decode(), F.fake_value(i)) for i in range(start, F.fake_calls())]
cfg = synth.TINY
weights = synth.make_model(cfg, seed=1)
"""


@pytest.fixture(scope="module")
def child(tmp_path_factory):
    """Runs Python code in a process whose CUDA runtime is the fake."""
    fake = str(tmp_path_factory.mktemp("fake") / "fake_cudart.so")
    cuda_home = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", f"-I{cuda_home}/include", os.path.join(HERE, "fake_cudart.c"), "-o",
                    fake], check=True)
    prelude = PRELUDE.format(pkg=os.path.join(os.path.dirname(HERE), "inferencer-jetson_b200"), fake=fake)

    def run(code):
        r = subprocess.run([sys.executable, "-c", prelude + code], env=dict(os.environ, LD_PRELOAD=fake),
                           capture_output=True, text=True, timeout=120)
        assert r.returncode == 0, r.stdout + r.stderr
    return run


@pytest.mark.parametrize("kv_type", [None, "f16", "e4m3"])
@pytest.mark.parametrize("fail", ["cudaEventRecord", "cudaMemcpyAsync", "cudaLaunchKernelExC"])
def test_a_sampled_step_that_fails_waits_for_what_it_started(child, fail, kv_type):
    """The step's graph reads pinned memory that the next step writes: every way out of the call waits for it."""
    child(f"""
e = Engine(cfg, weights, context=64, max_batch=4, max_seqs=2, kv_type={kv_type!r})
s = e.seq_open()
e.decode_sample([s], [3], [0.5])
start = F.fake_calls()
F.fake_fail(b"{fail}", b"cudaGraphLaunch")
try:
    e.decode_sample([s], [4], [0.5])
    raise SystemExit("no error")
except lib.IjbError as err:
    assert "made by the test" in str(err), err
calls = [n for n, _ in log(start)]
assert "cudaGraphLaunch" in calls
behind = calls[len(calls) - calls[::-1].index("cudaGraphLaunch"):]
assert "{fail}" in behind and "cudaStreamSynchronize" in behind[behind.index("{fail}"):], behind
assert e.seq_length(s) == 1
e.decode_sample([s], [4], [0.5])
assert e.seq_length(s) == 2
""")


@pytest.mark.parametrize("kv_type", ["f16", "e4m3"])
def test_paged_engines_take_no_memory_of_the_other_attention(child, kv_type):
    """Its partial records grow with max_batch times context; an engine whose attention is the paged one has none."""
    child(f"""
kw = dict(context=5000, max_batch=8, max_seqs=2)
records = 8 * cfg.heads * -(-5000 // 128) * (cfg.head_dim + 2) * 4 + 16  # an allocation's slack
e = Engine(cfg, weights, **kw)
assert ("cudaMalloc", records) in log()
start = F.fake_calls()
e = Engine(cfg, weights, kv_type={kv_type!r}, **kw)
assert ("cudaMalloc", records) not in log(start)
s = e.seq_open()
e.decode_step([s], [1])
assert e.time_layer_attention([s], reps=2)[1] == cfg.kv_heads * 2 * {{"f16": 2 * cfg.head_dim, "e4m3": cfg.head_dim + 1}}[{kv_type!r}]
""")


@pytest.mark.parametrize("largest", [16, 8])
def test_sampling_without_clusters_of_16(child, largest):
    """Few rows take clusters of 16, a size that a device (or a part of one) need not place: then 8, as many rows do."""
    child(f"""
L = lib.load()
F.fake_largest_cluster({largest})
for n, want in ((1, {largest}), (8, {largest}), (9, 8)):
    start = F.fake_calls()
    assert L.ijb_sample(4096, 128256, n, 128256, 4096, None, None, None, None, 4096, None, None) == 0
    assert [v for name, v in log(start) if name == "cudaLaunchKernelExC"] == [want]
""")


def test_attention_refuses_a_scale_beyond_its_base_2_logarithm(child):
    """Scores are scaled by scale * log2(e), which has to be a number too: an infinity makes NaN of a score of 0."""
    child("""
L = lib.load()
v = lib.KvView(type=2, kv_heads=2, head_dim=64, page_size=16, num_pages=4, data_dev=4096, scale_dev=8192,
               page_table_dev=256, n_seqs=1, max_pages=4)
def attention(scale):
    return L.ijb_paged_attention(ctypes.byref(v), 4, 0, 4096, 256, 8192, 256, 2, 1, 256, None, 256, 1, scale, 4096, 1 << 40,
                                 None, None)
assert attention(0.125) == lib.OK and attention(2e38) == lib.OK
for scale in (2.4e38, 3.4e38, float("inf"), 0.0, -1.0, float("nan")):
    assert attention(scale) == lib.ERR_INVALID and "scale" in L.ijb_last_error(None).decode()
""")
