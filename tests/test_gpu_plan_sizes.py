"""Plans around the sizes at which they change their form: one block of many experts or few, two launches, three."""
import pytest
import torch

from burn_automata_amd import experts
from tests.test_gpu_experts import check_plan

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("count", (510, 511, 512, 513, 777, 1024))
@pytest.mark.parametrize("entries", (0, 1, 64, 65, 511, 512, 513, 3585, 4095, 4096, 4097, 8192, 8193))
def test_plans_of_many_experts(entries, count):
    g = torch.Generator(device="cuda").manual_seed(entries + count)
    chosen = torch.randint(-1, count + 1, (entries, 1), generator=g, device="cuda", dtype=torch.int32)
    check_plan(experts.plan(chosen, count), chosen, count)
    few = torch.randint(count - 3, count + 1, (entries, 1), generator=g, device="cuda", dtype=torch.int32)
    check_plan(experts.plan(few, count), few, count)


@pytest.mark.parametrize("rows,count,k", ((1, 512, 8), (130, 1024, 31), (129, 700, 32)))
def test_routes_of_many_experts(rows, count, k):
    g = torch.Generator(device="cuda").manual_seed(rows)
    r = experts.route(torch.randn(rows, count, generator=g, device="cuda"), k)
    check_plan(r.plan, r.experts, count)
