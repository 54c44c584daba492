#define FTA_INST_D 128
#include "fta_token_stage1.inc"
