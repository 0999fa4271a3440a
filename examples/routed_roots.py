"""Vectors through their root codewords' own 8-bit projections, and one step of training on the exchange.

    python examples/routed_roots.py [--vectors 20000] [--roots 64] [--dim 128] [--out 96]

The large-root encoder assigns every vector to a root codeword.  The nearest other root by an 8-bit score joins as a second
choice, both weighted by a softmax of their scores.  The vectors are sorted by root, quantised into that order, taken
through each root's own projection in 8-bit integers, and brought back with the weights.  Then the same exchange in 32 bits
takes a gradient step on a scale for each root's rows and on the weights.  Needs a GPU.
"""
import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import stlq_b200  # noqa: E402


def main(vectors=20000, roots=64, dim=128, out_dim=96, seed=0):
    rng = np.random.default_rng(seed)
    centres = rng.uniform(0, 255, (roots, dim)).astype(np.float32)
    X = centres[rng.integers(0, roots, vectors)] + rng.normal(0, 25, (vectors, dim)).astype(np.float32)
    books = np.concatenate([centres, rng.normal(0, 25, (512, dim)).astype(np.float32)])
    x = torch.from_numpy(X).cuda()

    # The assignment, as the large pipeline makes it.
    enc = stlq_b200.Encoder(books, [roots, 256, 256], device=0, large_root=True)
    cluster = enc.encode_base_large_root_device(x, beam=4, icm_iters=0)[0].long()
    enc.sync()

    # A second choice: the best other root by 8-bit scores (of unit codewords, so that length does not decide).
    k = stlq_b200.Kernels(0)
    unit = torch.nn.functional.normalize(torch.from_numpy(centres).cuda(), dim=1)
    root_q, root_s = k.quantize_rows(unit)  # laid out once
    scores = k.matmul_i8(*k.quantize_rows(x), root_q, root_s, out_dtype=torch.float32)
    first = scores.gather(1, cluster[:, None])
    second = scores.scatter(1, cluster[:, None], float("-inf")).max(1)
    ids = torch.stack([cluster, second.indices], 1)
    mix = torch.softmax(torch.cat([first, second.values[:, None]], 1) / 50.0, 1)

    # Each root's projection in 8 bits, over its own rows.
    W = torch.randn(roots, out_dim, dim, generator=torch.Generator().manual_seed(seed)).cuda() / dim**0.5
    wq, ws = k.quantize_rows(W.flatten(0, 1))
    r = k.sort_by_expert(ids, roots)
    q, s = k.dispatch_i8(x, r)
    y = k.matmul_i8_grouped(q, s, wq.unflatten(0, (roots, out_dim)), ws.view(roots, out_dim), r.offsets, out_dtype=torch.float32)
    out = k.combine(y, mix, r)
    k.sync()
    want = sum(torch.bmm(W[ids[:, j]], x[..., None])[..., 0] * mix[:, j, None] for j in range(2))
    error = float((out - want).norm() / want.norm())
    print(f"{vectors} vectors, {roots} roots: rows per root {int(r.offsets.diff().min())} to {int(r.offsets.diff().max())}, "
          f"relative error of the 8-bit projections {error:.4f}")

    # One step on the same exchange in 32 bits: a scale for each root's rows, and the weights.
    expert_of_row = ids.reshape(-1)[r.order.long()]
    scale = torch.ones(roots, 1, device="cuda", requires_grad=True)
    logits = mix.log().requires_grad_()
    target = x * 1.05

    def loss():
        rows = k.dispatch(x, r) * scale[expert_of_row]
        return (k.combine(rows, torch.softmax(logits, 1), r) - target).square().mean()

    before = loss()
    before.backward()
    with torch.no_grad():
        scale -= 0.02 * scale.grad / scale.grad.norm()
        logits -= 0.02 * logits.grad / logits.grad.norm()
        before, after = float(before), float(loss())
    print(f"training step: loss {before:.4f} -> {after:.4f}")
    return error, before, after


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--vectors", type=int, default=20000)
    ap.add_argument("--roots", type=int, default=64)
    ap.add_argument("--dim", type=int, default=128)
    ap.add_argument("--out", type=int, default=96)
    a = ap.parse_args()
    main(a.vectors, a.roots, a.dim, a.out)
