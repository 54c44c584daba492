#define FTA_INST_D 64
#include "fta_token_stage1.inc"
