"""The package's names without torch, which only some of them need."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run(code):
    env = dict(os.environ, PYTHONPATH=os.path.join(ROOT, "moe-prefetch_amd"))
    p = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=120)
    assert p.returncode == 0, p.stderr
    return p.stdout.split()


def test_a_star_import_takes_no_torch():
    assert run("""
import sys
sys.modules["torch"] = None                           # an import of it fails
from moe_prefetch import *
print(MoeCache.__name__, ExpertCache.__name__, TYPE_Q4K)
""") == ["MoeCache", "ExpertCache", "12"]


def test_the_names_that_need_torch_are_there_by_name():
    assert run("""
import sys
import moe_prefetch
assert "torch" not in sys.modules
assert {"BlockNorm", "Sampler", "ScoredRouter"} <= set(dir(moe_prefetch))
from moe_prefetch import BlockNorm, Sampler, ScoredRouter
print(BlockNorm.__name__, Sampler.__name__, ScoredRouter.__name__)
""") == ["BlockNorm", "Sampler", "ScoredRouter"]
