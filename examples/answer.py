"""A model that answers: its Linears' weights in 4 bits, a prompt, one token at a time with the alternatives it had, and the score of a text.

    python examples/answer.py [--layers 2] [--hidden 1024] [--vocab 8192] [--tokens 16] [--batch 1]

The parameters are random: the text is none, the calls are those of a trained model."""
import argparse
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from pratchya_b200._nnx_impl import generate, score  # noqa: E402
from pratchya_b200._nnx_impl._model import PratchyaCausalLM, PratchyaConfig  # noqa: E402


def main():
    ap = argparse.ArgumentParser()
    for name, value in (("layers", 2), ("hidden", 1024), ("vocab", 8192), ("tokens", 16), ("batch", 1)):
        ap.add_argument("--" + name, type=int, default=value)
    a = ap.parse_args()
    model = PratchyaCausalLM(PratchyaConfig(vocab_size=a.vocab, hidden_size=a.hidden, intermediate_size=4 * a.hidden, n_layers=a.layers)).to_int4(group=64, zero_points=True)
    gen = torch.Generator(device="cuda").manual_seed(0)
    prompt = torch.randint(0, a.vocab, (a.batch, 12), generator=gen, device="cuda")
    generate(model, prompt, 2, top=5)
    torch.cuda.synchronize()
    began = time.perf_counter()
    answer = generate(model, prompt, a.tokens, top=5, uniform=torch.rand(a.batch, a.tokens, generator=gen, device="cuda"))
    torch.cuda.synchronize()
    print(f"{a.tokens} tokens for each of {a.batch} in {time.perf_counter() - began:.3f} s")
    for t, lp, h, tops in zip(answer.tokens[0].tolist(), answer.logprobs[0].tolist(), answer.entropy[0].tolist(), answer.top_tokens[0].tolist()):
        print(f"token {t:6d}  log probability {lp:7.3f}  entropy {h:6.3f}  best {tops}")
    with torch.no_grad():
        text = score(model, torch.cat([prompt, answer.tokens], dim=1), top=1)
    # read at once, not token by token as above: the norm over a block's heads runs over the tokens of a call, so these are other numbers than the answer's
    print(f"log probability of the whole text {float(text.logprobs[0].sum()):.2f} over {text.logprobs.shape[1]} tokens")


if __name__ == "__main__":
    main()
