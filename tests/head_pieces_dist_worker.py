"""tests/dist_worker.py with models that keep no logits."""
import functools

import dist_worker
from llmc_b200.models import gpt2, llama3

if __name__ == "__main__":
    gpt2.GPT = functools.partial(gpt2.GPT, head_pieces=True)
    llama3.Llama = functools.partial(llama3.Llama, head_pieces=True)
    dist_worker.main()
