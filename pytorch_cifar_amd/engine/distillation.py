"""Distillation in the training step: a frozen zoo model answers each batch, and the student learns
from its top logits beside the labels (``ops.distill``).

``main.py`` / ``main_dist.py``: ``--teacher NAME --teacher_ckpt PATH`` with ``--distill_k``,
``--distill_temp``, ``--distill_alpha`` and ``--distill_tail``. The logged loss and accuracy stay the
student's cross-entropy and hits on the labels, so runs with and without a teacher compare.
"""
from __future__ import annotations

import torch

from ..ops.distill import distill_loss, top_logits
from ..ops.functional import cross_entropy, enable_batched_weight_prep


class Distillation:
    """``teacher``: a model on the step's device; it is set to eval and its parameters are frozen.
    ``k`` of its logits are kept, at ``temperature``; ``alpha`` weighs its term against the labels';
    ``tail`` adds the mass it leaves to the other classes as one class (``ops.distill``)."""

    def __init__(self, teacher, k=5, temperature=4.0, alpha=0.9, tail=True):
        self.teacher = teacher.eval().requires_grad_(False)
        self.k, self.temperature, self.alpha, self.tail = k, temperature, alpha, tail
        p = next(teacher.parameters(), None)
        if p is not None and p.is_cuda:
            # its weights stand still: the bf16 operands are written once
            enable_batched_weight_prep(teacher).__dict__["_pca_wplan"].skip_when_fresh = True

    @torch.no_grad()
    def answer(self, x):
        """The teacher's top logits for a batch (before the student's forward: each model's operand
        plan is the current one during its own)."""
        return top_logits(self.teacher(x), self.k, self.temperature)

    def loss(self, logits, top, target, metrics=None):
        if metrics is not None:
            with torch.no_grad():
                cross_entropy(logits.detach(), target, metrics)
        return distill_loss(logits, top, target, temperature=self.temperature, alpha=self.alpha,
                            tail=self.tail)


def add_arguments(parser):
    parser.add_argument('--teacher', default=None, help='zoo model whose answers the net learns from')
    parser.add_argument('--teacher_ckpt', default=None, metavar='CKPT', help="the teacher's checkpoint")
    parser.add_argument('--distill_k', default=5, type=int, help="teacher's logits kept a sample")
    parser.add_argument('--distill_temp', default=4.0, type=float, help='distillation temperature')
    parser.add_argument('--distill_alpha', default=0.9, type=float,
                        help="weight of the teacher's term; the labels' is 1 - alpha")
    parser.add_argument('--distill_tail', default=1, type=int,
                        help='1: the mass of the other classes is one more term; 0: the kept logits alone')


def check_arguments(parser, args):
    if (args.teacher is None) != (args.teacher_ckpt is None):
        parser.error('--teacher and --teacher_ckpt go together')
    if args.teacher is not None:
        if not 1 <= args.distill_k <= 10:
            parser.error('--distill_k must be 1 to 10')
        if not args.distill_temp > 0 or not 0 <= args.distill_alpha <= 1:
            parser.error('--distill_temp must be positive and --distill_alpha in [0, 1]')


def from_arguments(args, device):
    """The run's :class:`Distillation`, or None. Every rank loads its own copy of the teacher."""
    if args.teacher is None:
        return None
    from .. import models
    from .checkpoint import load_checkpoint

    teacher = models.build_model(args.teacher).to(device)
    load_checkpoint(args.teacher_ckpt, teacher, map_location=device)
    return Distillation(teacher, args.distill_k, args.distill_temp, args.distill_alpha,
                        bool(args.distill_tail))
