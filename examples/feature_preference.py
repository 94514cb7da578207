"""Entity rows from features, trained by preference against a frozen model: features -> linear layers with dropout -> rows -> DistMult
scores against shared negatives -> preference loss relative to what the frozen model gives the same triples -> gradients -> updates.

    python examples/feature_preference.py [--steps 60]

The graph is synthetic: a triple (h, r, t) holds if t is the entity whose features lie nearest to the relation's rotation of h's.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from cuke_amd import FeatureEncoder, KGEModel, TrainSampler, inspect, preference_loss, sparse_adagrad  # noqa: E402

FEATURES, HIDDEN, DIM, CHUNK, NEGATIVES = 96, 256, 128, 64, 64


def make_graph(n_ent, n_rel, n_triples, seed, dev):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n_ent, FEATURES, generator=g)
    turn = torch.linalg.qr(torch.randn(n_rel, FEATURES, FEATURES, generator=g)).Q
    h, r = torch.randint(0, n_ent, (n_triples,), generator=g), torch.randint(0, n_rel, (n_triples,), generator=g)
    moved = (x[h].unsqueeze(1) @ turn[r]).squeeze(1)
    like = moved @ x.T
    like[torch.arange(n_triples), h] = -float("inf")
    return x.to(dev), tuple(v.numpy() for v in (h, r, like.argmax(1)))


def train(steps=60, n_ent=2000, n_rel=8, batch=512, dtype=torch.bfloat16, lr=0.05, drop=0.1, seed=0, dev="cuda:0"):
    """The loss of every step."""
    x, triples = make_graph(n_ent, n_rel, 8 * batch, seed, dev)
    x = x.to(dtype)
    g = torch.Generator().manual_seed(seed + 1)
    normal = lambda *shape, scale: (torch.randn(shape, generator=g) * scale).to(dev)
    master = [normal(HIDDEN, FEATURES, scale=FEATURES ** -0.5), torch.zeros(HIDDEN, device=dev), normal(DIM, HIDDEN, scale=HIDDEN ** -0.5),
              torch.zeros(DIM, device=dev)]                                       # fp32 weights, multiplied as `dtype`
    second = [torch.zeros_like(w) for w in master]
    E, R = normal(n_ent, DIM, scale=0.05), normal(n_rel, DIM, scale=0.3)          # free rows of the entities, and the relations
    state_e, state_r = torch.zeros(n_ent, device=dev), torch.zeros(n_rel, device=dev)
    encoder = FeatureEncoder(*(w.to(dtype) for w in master), act="gelu", drop=drop, row_drop=drop / 2, seed=seed)
    frozen = KGEModel("DistMult", encoder.encode(x, E), R.clone())               # the reference: the model as it starts
    losses = []
    sampler = TrainSampler(triples, n_ent, batch, NEGATIVES, CHUNK, seed=seed, device=dev)
    for step in range(steps):
        h, r, t, neg = next(sampler)
        entities = inspect([h, t, neg], n_ent)                                   # every entity of the batch is encoded once
        ids, at = entities.ids(), entities.inverse.long()
        fw = encoder.forward(x[ids], E[ids], step=step)
        model = KGEModel("DistMult", fw.rows, R)
        scores = model.score(at[:batch], r, at[batch:2 * batch], at[2 * batch:], CHUNK)
        ref = frozen.score(h, r, t, neg, CHUNK)
        # (a negative that is the positive's own tail is no negative)
        mask = neg.view(-1, 1, NEGATIVES) != t.view(-1, CHUNK, 1)
        loss, dpos, dneg = preference_loss(scores.pos, scores.neg, ref.pos, ref.neg, beta=0.5, smoothing=0.01, temperature=0.5,
                                           mask=mask.view(batch, NEGATIVES))
        grads = model.backward(scores, dpos, dneg)                               # every row of the batch occurs: ids are 0 .. n - 1
        back = encoder.backward(fw, grads.ent_rows)
        sparse_adagrad(E, state_e, entities, back.base, lr)
        sparse_adagrad(R, state_r, scores.rel_insp, grads.rel_rows, lr)
        for w, s, d in zip(master, second, (back.hidden.weight, back.hidden.bias, back.last.weight, back.last.bias)):
            d = d.float()
            s.add_(d * d)
            w.addcdiv_(d, s.sqrt().add_(1e-10), value=-lr)
        encoder.w1, encoder.b1, encoder.w2, encoder.b2 = (w.to(dtype) for w in master)
        losses.append(loss)
    return torch.cat(losses).tolist()


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=60)
    a = ap.parse_args()
    out = train(a.steps)
    for i in range(0, len(out), max(1, len(out) // 10)):
        print(f"step {i:4d}  loss {out[i]:.4f}")
    print(f"step {len(out) - 1:4d}  loss {out[-1]:.4f}")
