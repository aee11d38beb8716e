"""k_az_step, one search a lane: searches of one wave that leave a step at different
rounds, for different reasons, each as if it ran alone (csrc/os_az.h az_step)."""
import numpy as np
import pytest

import oracle_lib
from os_amd import engine as E
from test_az import _gpu_toy_evaluator, _oracle_eval_fn


@pytest.mark.gpu
@pytest.mark.parametrize("requests", ["separate", "fused"])
@pytest.mark.parametrize("puct", [True, False])
@pytest.mark.parametrize("game,plies", [("tic_tac_toe", 6), ("connect_four", 30),
                                        ("breakthrough(rows=6,columns=6)", 20),
                                        ("hex(board_size=4)", 11), ("hex(board_size=5)", 8),
                                        ("go(board_size=5)", 12)])
def test_gpu_lanes_leave_a_step_apart(require_gpu, game, plies, puct, requests):
  """Roots at many depths, near the game's end among them: proven roots stop early,
  terminal leaves take further simulations within a step, inner nodes ask for
  priors while their neighbours ask for values."""
  from os_amd.az import ExternalEvaluatorSearch
  R, sims = 70, 20
  acts, offs = E.make_roots(game, R, seed_base=11, max_plies=plies)
  seeds = np.arange(R, dtype=np.uint32) * 7 + 3
  og = oracle_lib.Game(game)
  A = og.num_distinct_actions
  kw = dict(puct=puct, uct_c=1.5, max_simulations=sims)
  ref = og.mcts_external(acts, offs, seeds, _oracle_eval_fn(game), max_children=A, **kw)
  search = ExternalEvaluatorSearch(game)
  got = search.run(acts, offs, seeds, _gpu_toy_evaluator(A), requests=requests, layout="lane", **kw)
  mc = search.eng.max_children
  for k in E.OUTPUT_KEYS:
    r = ref[k][:, :mc] if ref[k].ndim == 2 else ref[k]
    bad = np.nonzero((got[k] != r).reshape(R, -1).any(axis=1))[0]
    assert bad.size == 0, (k, bad.tolist())
