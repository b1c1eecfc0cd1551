"""Post-training a small selective state space language model on one GPU.

Each step samples responses to a batch of ragged prompts token by token
(causal_conv_step, selective_scan_step), scores them in one pass over the
whole sequences (causal_conv, selective_scan, token_logprobs) and updates the
model with the clipped policy loss; a preference step on pairs of responses
follows.  The reward is synthetic: the share of even token ids.

    python examples/posttrain_selective_lm.py --steps 5
"""
import argparse
import copy
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
import mogt_b200  # noqa: E402
from mogt_b200.selective_lm import SelectiveLM  # noqa: E402


@torch.no_grad()
def sample(model, prompts, lengths, new_tokens, generator):
    """[B, new_tokens] sampled continuations of the prompts' first `lengths` tokens."""
    logits, caches = model.prefill(prompts, lengths)
    out = []
    for _ in range(new_tokens):
        tok = torch.multinomial(torch.softmax(logits.float(), -1), 1, generator=generator)[:, 0]
        out.append(tok)
        logits = model.step(tok, caches)
    return torch.stack(out, 1)


def assemble(prompts, lengths, responses):
    """Sequences [prompt, response, padding], labels (the next token) and the
    mask of the labels that belong to the response."""
    B, P = prompts.shape
    R = responses.shape[1]
    ids = prompts.new_zeros(B, P + R)
    ids[:, :P] = prompts
    at = lengths[:, None] + torch.arange(R, device=ids.device)[None]
    ids.scatter_(1, at, responses)
    labels = torch.full_like(ids, -100)
    labels[:, :-1] = ids[:, 1:]
    pos = torch.arange(P + R, device=ids.device)[None]
    mask = (pos >= lengths[:, None] - 1) & (pos < lengths[:, None] + R - 1)
    return ids, labels, mask


def reward(responses):
    return (responses % 2 == 0).float().mean(1)


def main(argv=None):
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=5)
    ap.add_argument("--batch", type=int, default=16)
    ap.add_argument("--prompt", type=int, default=24)
    ap.add_argument("--new-tokens", type=int, default=32)
    ap.add_argument("--vocab", type=int, default=512)
    ap.add_argument("--d-model", type=int, default=128)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--lr", type=float, default=2e-3)
    ap.add_argument("--seed", type=int, default=0)
    args = ap.parse_args(argv)
    torch.manual_seed(args.seed)
    gen = torch.Generator(device="cuda").manual_seed(args.seed)
    model = SelectiveLM(args.vocab, args.d_model, args.layers).cuda()
    reference = copy.deepcopy(model).eval()
    opt = torch.optim.AdamW(model.parameters(), lr=args.lr)
    history = []
    for step in range(args.steps):
        prompts = torch.randint(0, args.vocab, (args.batch, args.prompt), generator=gen, device="cuda")
        lengths = torch.randint(1, args.prompt + 1, (args.batch,), generator=gen, device="cuda")
        responses = sample(model, prompts, lengths, args.new_tokens, gen)
        ids, labels, mask = assemble(prompts, lengths, responses)
        r = reward(responses)
        advantages = (r - r.mean()) / (r.std() + 1e-4)
        with torch.no_grad():
            old = mogt_b200.token_logprobs(model(ids), labels, mask=mask)
            ref = mogt_b200.token_logprobs(reference(ids), labels, mask=mask)
        for _ in range(2):
            loss = mogt_b200.policy_loss(model(ids), labels, old, advantages, ref_logprobs=ref, mask=mask, kl_coef=0.02)
            opt.zero_grad()
            loss.backward()
            opt.step()
        # pairs: the better half of the batch against the worse half
        order = torch.argsort(r, descending=True)
        order = order[:2 * (args.batch // 2)]
        pref = mogt_b200.preference_loss(model(ids[order]), labels[order], ref.double().sum(1)[order], beta=0.1,
                                         mask=mask[order])
        opt.zero_grad()
        pref.backward()
        opt.step()
        history.append(dict(reward=float(r.mean()), policy=float(loss.detach()), preference=float(pref.detach())))
        print(f"step {step}: reward {history[-1]['reward']:.3f}  policy loss {history[-1]['policy']:+.4f}  "
              f"preference loss {history[-1]['preference']:.4f}")
    return history


if __name__ == "__main__":
    main()
