#!/bin/bash
# Round 5, GPU call I: the production library with the extension units on the basic VGPR allocator: matrix, the whole GPU suite, stress
O=gpurun_out/r05i; mkdir -p $O
timeout 600 python scripts/gpu_matrix.py > $O/matrix_prod.txt 2>&1; tail -3 $O/matrix_prod.txt | cut -c1-300
timeout 1500 python -m pytest tests -m gpu -q > $O/pytest_gpu.txt 2>&1; echo "pytest rc $?" >> $O/pytest_gpu.txt; tail -6 $O/pytest_gpu.txt | cut -c1-300
timeout 600 python scripts/stress_cfgs.py env,ms,cfg1,anim,b8 40 > $O/stress_prod.txt 2>&1; tail -2 $O/stress_prod.txt | cut -c1-300
