"""The command line's scores and drafts."""
import os
import subprocess
import sys

import pytest

from tiny_models import CONFIGS, prompt, write_model

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run(*args):
    p = subprocess.run([sys.executable, "-m", "rocml_b200", *args], cwd=ROOT, capture_output=True, text=True, timeout=300)
    return p.returncode, p.stdout, p.stderr


def test_scores_and_drafts(tmp_path):
    folder = str(tmp_path)
    write_model(folder, CONFIGS["B"], seed=41, std=0.08)
    ids = prompt(5, 21, CONFIGS["B"]["vocab_size"])
    text = ",".join(map(str, ids))
    common = ["--model", folder, "--dtype", "float32", "--ctx", "128"]
    rc, out, err = run("score", *common, "--prompt-ids", text, "--top", "2")
    assert rc == 0, err
    lines = out.strip().splitlines()
    assert [int(x.split()[0]) for x in lines] == ids[1:] and all(x.count(":") == 2 for x in lines) and "perplexity" in err
    rc, plain, err = run("generate", *common, "--prompt-ids", text, "-n", "12", "--logprobs", "3")
    assert rc == 0, err
    tokens = plain.splitlines()[0].split()
    assert [x.split()[0] for x in plain.splitlines()[1:]] == tokens
    rc, drafted, err = run("generate", *common, "--prompt-ids", text, "-n", "12", "--draft", "4")
    assert rc == 0 and drafted.split() == tokens, err
    rc, _, err = run("generate", *common, "--prompt-ids", text, "-n", "3", "--logprobs", "40")
    assert rc == 1 and "alternatives" in err
