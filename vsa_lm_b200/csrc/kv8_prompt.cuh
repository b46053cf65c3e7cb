// The attention kernel for many query rows (kv8_prompt.cu), which bolt3_kv8_attend calls.
#pragma once

#include "../../include/bolt3.h"
#include "kv8.cuh"

size_t kv8_prompt_workspace(int B, int T, int H, int HKV, int HD, int64_t n);
int kv8_prompt_launch(const bolt3_kv8_attend_args* a, const kv8::Length& len, cudaStream_t s);
